// cafe_interact.hip -- DLRM's dot interaction (dlrm_s_pytorch.py:779-809): a sample's nf feature rows t_0 .. t_{nf-1}
// (the bottom MLP's output first, if there is one, then one embedding row per field), every pair's inner product
//
//     out = [t_0 (with dense features) | <t_i, t_j> for i = 0 .. nf-1, j = 0 .. i-1 (.. i with `itself`)]
//     dt_i = sum_j s_ij t_j,  s_ij = s_ji the pair's gradient (s_ii twice it), and dt_0 += the gradient of its copy
//
// Embedding rows come as the collection writes them, [F, B, D].  One wave per sample; products on the float32 matrix
// units (16 x 16 x 4), whatever the rows' types.
#include "cafe_dense.h"

#include <algorithm>

using namespace cafe;

namespace {

struct InteractArgs {
    const void *x; int64_t ldx;                     // [B, D] or null
    const void *emb; int64_t sf, sb;                // [F, B, D]: strides of field and sample
    void *out; int64_t ldo;
    const void *dout; int64_t lddo;
    void *dx; int64_t lddx;
    void *demb; int64_t dsf, dsb;
    int64_t B;
    int F, D, nf, pairs, itself, lead;              // lead: D with dense features, else 0
};

__device__ __forceinline__ int pair_at(int i, int j, int itself) { return (itself ? i * (i + 1) / 2 : i * (i - 1) / 2) + j; }

// four elements at p as floats, zeros from element n on
template <class T> __device__ __forceinline__ f32x4 load4(const T *p, int n) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) {
            v = __builtin_bit_cast(f32x4, load16(p));
        } else {
            struct __attribute__((packed, aligned(2))) Half { u32x2 v; };
            union { u32x2 v; T e[4]; } u;
            u.v = ((const Half *)p)->v;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = (float)u.e[e];
        }
        return v;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < n) v[e] = (float)p[e];
    return v;
}
template <class T> __device__ __forceinline__ void store4(T *p, f32x4 v, int n) {
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) {
            store16(p, __builtin_bit_cast(u32x4, v));
        } else {
            struct __attribute__((packed, aligned(2))) Half { u32x2 v; };
            union { u32x2 v; T e[4]; } u;
#pragma unroll
            for (int e = 0; e < 4; e++) u.e[e] = (T)v[e];
            ((Half *)p)->v = u.v;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (e < n) p[e] = (T)v[e];
}

template <class TE, class T> __device__ __forceinline__ f32x4 load_row(const InteractArgs &g, int64_t b, int row, int d) {
    if (row >= g.nf) return f32x4{0.f, 0.f, 0.f, 0.f};
    if (g.lead) {
        if (row == 0) return load4((const T *)g.x + b * g.ldx + d, g.D - d);
        row--;
    }
    return load4((const TE *)g.emb + row * g.sf + b * g.sb + d, g.D - d);
}

// RT tiles of 16 rows.  Lane l holds row l % 16 of each tile, four consecutive d from 4 (l / 16): with the reduction
// renumbered alike on both sides that is A's and B's fragment at once, so a tile is loaded once for all its products.
template <class TE, class T, int RT> __global__ __launch_bounds__(256) void k_interact(InteractArgs g) {
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    for (int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); b < g.B; b += (int64_t)gridDim.x * 4) {
        f32x4 acc[RT * (RT + 1) / 2];
#pragma unroll
        for (int i = 0; i < RT * (RT + 1) / 2; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int d0 = 0; d0 < g.D; d0 += 16) {
            f32x4 t[RT];
#pragma unroll
            for (int i = 0; i < RT; i++) t[i] = load_row<TE, T>(g, b, 16 * i + r, d0 + 4 * q);
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int j = 0; j <= i; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        acc[i * (i + 1) / 2 + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(t[i][e], t[j][e], acc[i * (i + 1) / 2 + j], 0, 0, 0);
        }
        T *out = (T *)g.out + b * g.ldo;
        if (g.lead)
            for (int d = lane; d < g.D; d += 64) out[d] = ((const T *)g.x)[b * g.ldx + d];
        // accumulator element e of lane l: row 4 (l / 16) + e, column l % 16
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int j = 0; j <= i; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int row = 16 * i + 4 * q + e, col = 16 * j + r;
                    if (row < g.nf && col < row + g.itself) out[g.lead + pair_at(row, col, g.itself)] = (T)acc[i * (i + 1) / 2 + j][e];
                }
    }
}

// The pairs' gradients of a sample are staged in LDS (each is used twice).  Product S T: A is S (row l % 16, k = l / 16),
// B's column l % 16 stands for d = 64 u + 4 (l % 16) + e in product e, so that both T's loads and the results are four
// consecutive d per lane.
template <class TE, class T, int RT> __global__ __launch_bounds__(256) void k_interact_bwd(InteractArgs g) {
    extern __shared__ float lds[];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    float *s = lds + (threadIdx.x >> 6) * g.pairs;
    for (int64_t b0 = (int64_t)blockIdx.x * 4; b0 < g.B; b0 += (int64_t)gridDim.x * 4) {
        const int64_t b = b0 + (threadIdx.x >> 6);
        const T *dout = (const T *)g.dout + b * g.lddo;
        __syncthreads();
        if (b < g.B)
            for (int p = lane; p < g.pairs; p += 64) s[p] = (float)dout[g.lead + p];
        __syncthreads();
        if (b >= g.B) continue;
        const int steps = (g.nf + 3) >> 2;
        for (int d0 = 0; d0 < g.D; d0 += 64) {
            const int d = d0 + 4 * r;
            f32x4 acc[RT][4];
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i][e] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int k = 0; k < steps; k++) {
                const int j = 4 * k + q;
                const f32x4 t = load_row<TE, T>(g, b, j, d);
#pragma unroll
                for (int i = 0; i < RT; i++) {
                    const int row = 16 * i + r;
                    float a = 0.f;
                    if (row < g.nf && j < g.nf) {
                        if (row != j) a = s[row > j ? pair_at(row, j, g.itself) : pair_at(j, row, g.itself)];
                        else if (g.itself) a = 2.f * s[pair_at(row, row, 1)];
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, t[e], acc[i][e], 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < RT; i++)
#pragma unroll
                for (int v = 0; v < 4; v++) {
                    int row = 16 * i + 4 * q + v;
                    if (row >= g.nf || d >= g.D) continue;
                    f32x4 w = {acc[i][0][v], acc[i][1][v], acc[i][2][v], acc[i][3][v]};
                    if (g.lead) {
                        if (row == 0) {
                            if (g.dx) {
                                w += load4(dout + d, g.D - d);
                                store4((T *)g.dx + b * g.lddx + d, w, g.D - d);
                            }
                            continue;
                        }
                        row--;
                    }
                    if (g.demb) store4((TE *)g.demb + row * g.dsf + b * g.dsb + d, w, g.D - d);
                }
        }
    }
}

bool bad(const char *who, const InteractArgs &g, int te, int t) {
    if (g.B < 0 || g.F < 0 || g.D < 0) { set_error("%s: negative size", who); return true; }
    if (te < kF32 || te > kF16 || t < kF32 || t > kF16 || (te != kF32 && te != t)) {
        set_error("%s: type codes %d, %d (embedding rows are float32 or of the output's type)", who, te, t);
        return true;
    }
    if (g.nf > 128 || g.nf < 1) { set_error("%s: %d feature rows, 1 .. 128 expected", who, g.nf); return true; }
    return false;
}

template <class F> int by_types(int te, int t, F f) {
    if (te == kF32) {
        if (t == kF32) return f((float *)0, (float *)0);
        if (t == kBF16) return f((float *)0, (__bf16 *)0);
        return f((float *)0, (_Float16 *)0);
    }
    if (t == kBF16) return f((__bf16 *)0, (__bf16 *)0);
    return f((_Float16 *)0, (_Float16 *)0);
}

template <class TE, class T> int run_fwd(const InteractArgs &g, hipStream_t st) {
    const unsigned blocks = (unsigned)std::min<int64_t>((g.B + 3) / 4, 256 * 64);
#define CAFE_I(R) hipLaunchKernelGGL((k_interact<TE, T, R>), dim3(blocks), dim3(256), 0, st, g)
    if (g.nf <= 16) CAFE_I(1);
    else if (g.nf <= 32) CAFE_I(2);
    else if (g.nf <= 64) CAFE_I(4);
    else CAFE_I(8);
#undef CAFE_I
    CAFE_HIP_CHECK(hipGetLastError());
    return 0;
}
template <class TE, class T> int run_bwd(const InteractArgs &g, hipStream_t st) {
    const unsigned blocks = (unsigned)std::min<int64_t>((g.B + 3) / 4, 256 * 64);
    const size_t lds = (size_t)4 * g.pairs * 4;             // at most 4 waves x 128 * 129 / 2 floats = 132 KB
#define CAFE_I(R) do {                                                                                               \
        if (lds > 65536) CAFE_HIP_CHECK(hipFuncSetAttribute((const void *)k_interact_bwd<TE, T, R>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds)); \
        hipLaunchKernelGGL((k_interact_bwd<TE, T, R>), dim3(blocks), dim3(256), lds, st, g); } while (0)
    if (g.nf <= 16) CAFE_I(1);
    else if (g.nf <= 32) CAFE_I(2);
    else if (g.nf <= 64) CAFE_I(4);
    else CAFE_I(8);
#undef CAFE_I
    CAFE_HIP_CHECK(hipGetLastError());
    return 0;
}

}  // namespace

extern "C" int cafe_interact_fwd_dev(const void *d_x, int64_t ldx, const void *d_emb, int64_t field_stride, int64_t batch_stride, int64_t batch,
                                     int fields, int dim, int itself, int emb_dtype, int dtype, void *d_out, int64_t ldo, cafe_stream_t stream) {
    InteractArgs g = {};
    g.x = d_x; g.ldx = ldx; g.emb = d_emb; g.sf = field_stride; g.sb = batch_stride; g.out = d_out; g.ldo = ldo;
    g.B = batch; g.F = fields; g.D = dim; g.itself = itself ? 1 : 0;
    if (fields < 0 || fields > 128) { set_error("cafe_interact_fwd_dev: %d fields", fields); return 1; }
    g.nf = fields + (d_x ? 1 : 0); g.lead = d_x ? dim : 0;
    g.pairs = g.itself ? g.nf * (g.nf + 1) / 2 : g.nf * (g.nf - 1) / 2;
    if (bad("cafe_interact_fwd_dev", g, emb_dtype, dtype)) return 1;
    if (ldx < 0 || field_stride < 0 || batch_stride < 0 || ldo < (int64_t)g.lead + g.pairs) { set_error("cafe_interact_fwd_dev: bad stride"); return 1; }
    if (batch == 0 || g.lead + g.pairs == 0) return 0;
    if (!d_out || (fields > 0 && dim > 0 && !d_emb)) { set_error("cafe_interact_fwd_dev: null pointer"); return 1; }
    const hipStream_t st = (hipStream_t)stream;
    return by_types(emb_dtype, dtype, [&](auto te, auto t) {
        return run_fwd<std::remove_pointer_t<decltype(te)>, std::remove_pointer_t<decltype(t)>>(g, st); });
}

extern "C" int cafe_interact_bwd_dev(const void *d_dout, int64_t lddo, const void *d_x, int64_t ldx, const void *d_emb, int64_t field_stride,
                                     int64_t batch_stride, int64_t batch, int fields, int dim, int itself, int emb_dtype, int dtype, void *d_dx,
                                     int64_t lddx, void *d_demb, int64_t dfield_stride, int64_t dbatch_stride, cafe_stream_t stream) {
    InteractArgs g = {};
    g.x = d_x; g.ldx = ldx; g.emb = d_emb; g.sf = field_stride; g.sb = batch_stride; g.dout = d_dout; g.lddo = lddo;
    g.dx = d_dx; g.lddx = lddx; g.demb = d_demb; g.dsf = dfield_stride; g.dsb = dbatch_stride;
    g.B = batch; g.F = fields; g.D = dim; g.itself = itself ? 1 : 0;
    if (fields < 0 || fields > 128) { set_error("cafe_interact_bwd_dev: %d fields", fields); return 1; }
    g.nf = fields + (d_x ? 1 : 0); g.lead = d_x ? dim : 0;
    g.pairs = g.itself ? g.nf * (g.nf + 1) / 2 : g.nf * (g.nf - 1) / 2;
    if (bad("cafe_interact_bwd_dev", g, emb_dtype, dtype)) return 1;
    if (lddo < 0 || ldx < 0 || field_stride < 0 || batch_stride < 0 || dfield_stride < 0 || (d_dx && lddx < dim) || (d_demb && dbatch_stride < dim)) {
        set_error("cafe_interact_bwd_dev: bad stride");
        return 1;
    }
    if (d_dx && !d_x) { set_error("cafe_interact_bwd_dev: a gradient of dense features that are not there"); return 1; }
    if (batch == 0 || dim == 0 || (!d_dx && !d_demb)) return 0;
    if ((fields > 0 && !d_emb) || (g.lead + g.pairs > 0 && !d_dout)) { set_error("cafe_interact_bwd_dev: null pointer"); return 1; }
    const hipStream_t st = (hipStream_t)stream;
    return by_types(emb_dtype, dtype, [&](auto te, auto t) {
        return run_bwd<std::remove_pointer_t<decltype(te)>, std::remove_pointer_t<decltype(t)>>(g, st); });
}
