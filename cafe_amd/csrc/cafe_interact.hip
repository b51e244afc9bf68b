// cafe_interact.hip -- DLRM's dot interaction (dlrm_s_pytorch.py:779-809): a sample's nf feature rows t_0 .. t_{nf-1}
// (the bottom MLP's output first, if there is one, then one embedding row per field), every pair's inner product
//
//     out = [t_0 (with dense features) | <t_i, t_j> for i = 0 .. nf-1, j = 0 .. i-1 (.. i with `itself`)]
//     dt_i = sum_j s_ij t_j,  s_ij = s_ji the pair's gradient (s_ii twice it), and dt_0 += the gradient of its copy
//
// Embedding rows come as the collection writes them, [F, B, D].  One wave per sample; products on the float32 matrix
// units (16 x 16 x 4), whatever the rows' types.
#include "cafe_dense.h"

#include <type_traits>

using namespace cafe;

namespace {

struct InteractArgs {
    const void *x; int64_t ldx;                     // [B, D] or null
    const void *emb; int64_t sf, sb;                // [F, B, D]: strides of field and sample
    void *out; int64_t ldo;
    const void *dout; int64_t lddo;
    void *dx; int64_t lddx;
    void *demb; int64_t dsf, dsb;
    int64_t B, b0;                                  // samples b0 .. B - 1 are this launch's
    int F, D, nf, pairs, itself, lead;              // lead: D with dense features, else 0
};

__device__ __forceinline__ int pair_at(int i, int j, int itself) { return (itself ? i * (i + 1) / 2 : i * (i - 1) / 2) + j; }

// N consecutive elements (1, 2 or 4), at element alignment
template <class T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Run { T e[N]; };

// the first n of N elements at p as floats, zeros behind; nothing past them is read
template <class T, int N> __device__ __forceinline__ void load_run(const T *p, int n, float *v) {
    if (n >= N) {
        const Run<T, N> u = *(const Run<T, N> *)p;
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = (float)u.e[e];
        return;
    }
#pragma unroll
    for (int e = 0; e < N; e++) v[e] = e < n ? (float)p[e] : 0.f;
}
template <class T, int N> __device__ __forceinline__ void store_run(T *p, const float *v, int n) {
    Run<T, N> u;
#pragma unroll
    for (int e = 0; e < N; e++) u.e[e] = (T)v[e];
    if (n >= N) { *(Run<T, N> *)p = u; return; }
#pragma unroll
    for (int e = 0; e < N; e++)
        if (e < n) p[e] = u.e[e];
}

// One chunk of x as a chunk of the embedding rows' type.
template <class TE, class T> __device__ __forceinline__ u32x4 x_chunk(const T *p, int n) {
    if constexpr (sizeof(TE) == sizeof(T)) {
        return load_some(p, n);
    } else {
        float v[4];
        load_run<T, 4>(p, n, v);
        return u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
    }
}

__device__ __forceinline__ void wave_sync() {           // LDS written by this wave, read by other lanes of it
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One wave per sample, RT tiles of 16 rows.  Lane l loads row l % 16 of each tile, chunk l / 16 of the step's four: A's and
// B's fragment at once, so that a row is read once for all its products.  Rows behind the last one repeat it; their
// products are not stored.  U steps are requested together.  The pairs go through LDS, so that a sample's result leaves in
// 16-byte stores (RT = 8, which would leave one workgroup per compute unit, stores them as they are).  Bound by memory:
// 8192 x 27 x 128 in float32 takes 33.3 us (129 MB, 3.9 TB/s), 16384 x 27 x 16 with bfloat16 results 13.1 (41 MB, 3.1 TB/s).
template <class TE, class T, int RT> __global__ __launch_bounds__(256) void k_interact(InteractArgs g) {
    constexpr int E = Elem<TE>::per_chunk, ET = Elem<T>::per_chunk, STEP = 4 * E, U = RT <= 2 ? 4 : RT <= 4 ? 2 : 1;
    extern __shared__ float lds[];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int64_t b = g.b0 + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (b >= g.B) return;
    const bool isx = g.lead && r == 0;                  // row 0 of tile 0
    const T *px = (const T *)g.x + b * g.ldx;
    const TE *p[RT];
#pragma unroll
    for (int i = 0; i < RT; i++) {
        int row = 16 * i + r;
        row = (row < g.nf ? row : g.nf - 1) - (g.lead ? 1 : 0);
        p[i] = g.F ? (const TE *)g.emb + (row < 0 ? 0 : row) * g.sf + b * g.sb + q * E : nullptr;
    }
    f32x4 acc[RT * (RT + 1) / 2];
#pragma unroll
    for (int i = 0; i < RT * (RT + 1) / 2; i++) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const u32x4 (&t)[RT]) {
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int j = 0; j <= i; j++) acc[i * (i + 1) / 2 + j] = mfma16<TE>(t[i], t[j], acc[i * (i + 1) / 2 + j]);
    };
    int d = 0;
    if (g.F)
        for (; d + U * STEP <= g.D; d += U * STEP) {
            u32x4 t[U][RT];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < RT; i++) t[u][i] = load16(p[i] + d + u * STEP);
            if (isx) {
#pragma unroll
                for (int u = 0; u < U; u++) t[u][0] = x_chunk<TE, T>(px + d + u * STEP + q * E, E);
            }
#pragma unroll
            for (int u = 0; u < U; u++) multiply(t[u]);
        }
    if (g.F)
        for (; d + STEP <= g.D; d += STEP) {
            u32x4 t[RT];
#pragma unroll
            for (int i = 0; i < RT; i++) t[i] = load16(p[i] + d);
            if (isx) t[0] = x_chunk<TE, T>(px + d + q * E, E);
            multiply(t);
        }
    for (; d < g.D; d += STEP) {
        const int left = g.D - d - q * E;
        u32x4 t[RT];
#pragma unroll
        for (int i = 0; i < RT; i++) t[i] = g.F ? load_some(p[i] + d, left) : u32x4{0, 0, 0, 0};
        if (isx) t[0] = x_chunk<TE, T>(px + d + q * E, left);
        multiply(t);
    }
    T *out = (T *)g.out + b * g.ldo;
    for (int c = lane * ET; c < g.lead; c += 64 * ET) store_some(out + c, load_some(px + c, g.lead - c), g.lead - c);
    out += g.lead;
    float *s = lds + (threadIdx.x >> 6) * g.pairs;
#pragma unroll
    for (int i = 0; i < RT; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int row = 16 * i + 4 * q + e, at = pair_at(row, 0, g.itself);
#pragma unroll
            for (int j = 0; j <= i; j++) {
                const int col = 16 * j + r;
                if (row < g.nf && col < row + g.itself) {
                    if (RT == 8) out[at + col] = (T)acc[i * (i + 1) / 2 + j][e];
                    else s[at + col] = acc[i * (i + 1) / 2 + j][e];
                }
            }
        }
    if (RT == 8) return;
    wave_sync();
    for (int c = lane * ET; c < g.pairs; c += 64 * ET) {
        float v[ET];
#pragma unroll
        for (int e = 0; e < ET; e++) v[e] = c + e < g.pairs ? s[c + e] : 0.f;
        store_some(out + c, pack<T>(v), g.pairs - c);
    }
}

// dT = S T, one wave per sample.  The pairs' gradients are unfolded to the symmetric S in LDS (rows an odd number of words
// apart), where A's fragments (row l % 16, k = l / 16) are one read each: picked out of the flat list, their index
// arithmetic took longer than the products.  B's column l % 16 stands for d = VE (l % 16) + e in product e, so that T's
// loads and the results are VE neighbours per lane: 4, or fewer where 64 columns would stay empty.  One step's rows at a time
// up to 32 rows: enough waves are resident to keep memory busy (8192 x 27 x 128 in float32 takes 51.8 us, 54.6 with four
// steps' rows requested together); above, registers leave few waves and four steps go together (41 rows: 30.7 and 26.0).
// Bound by memory: those 242 MB pass at 4.6 TB/s, a large copy's rate.
template <class TE, class T, int RT, int VE, int WAVES> __global__ __launch_bounds__(WAVES * 64) void k_interact_bwd(InteractArgs g) {
    extern __shared__ float lds[];
    const int lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int64_t b = g.b0 + (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
    if (b >= g.B) return;
    constexpr int KB = RT <= 2 ? 1 : 4;                 // steps requested together
    const int stride = g.nf | 1, self = g.itself;
    float *s = lds + (threadIdx.x >> 6) * (g.nf * stride);
    const T *dout = (const T *)g.dout + b * g.lddo;
    for (int p0 = lane; p0 < g.pairs; p0 += 64 * 8) {
        float v[8];                                     // requested together
#pragma unroll
        for (int u = 0; u < 8; u++) v[u] = (float)dout[g.lead + (p0 + 64 * u < g.pairs ? p0 + 64 * u : g.pairs - 1)];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int p = p0 + 64 * u;
            if (p >= g.pairs) break;
            int i = (int)((__builtin_amdgcn_sqrtf((float)(8 * p + 1)) + (float)(1 - 2 * self)) * 0.5f);    // off by one at most
            if (pair_at(i, 0, self) > p) i--;
            if (pair_at(i + 1, 0, self) <= p) i++;
            const int j = p - pair_at(i, 0, self);
            s[i * stride + j] = i == j ? 2.f * v[u] : v[u];
            if (i != j) s[j * stride + i] = v[u];
        }
    }
    if (!self)
        for (int i = lane; i < g.nf; i += 64) s[i * stride + i] = 0.f;
    wave_sync();
    const int steps = (g.nf + 3) >> 2;
    const TE *emb = (const TE *)g.emb + b * g.sb;
    const float *mine[RT];                              // S's rows 16 i + l % 16
#pragma unroll
    for (int i = 0; i < RT; i++) mine[i] = s + (16 * i + r < g.nf ? 16 * i + r : 0) * stride;
    for (int d0 = 0; d0 < g.D; d0 += 16 * VE) {
        const int d = d0 + VE * r, left = g.D - d;
        f32x4 acc[RT][VE];
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int e = 0; e < VE; e++) acc[i][e] = f32x4{0.f, 0.f, 0.f, 0.f};
        // T(4 k + l / 16, d ..): the embedding rows, zeros in the place of x and behind the last.  FULL: loads are clamped, so
        // that none hangs on a lane's row and all of a step's are on their way together.
        auto rows = [&](int k, float (&t)[VE], auto fullc) {
            const int row = 4 * k + q - (g.lead ? 1 : 0);
            const bool there = row >= 0 && row < g.F;
            if constexpr (decltype(fullc)::value) {
                load_run<TE, VE>(emb + (row < 0 ? 0 : row < g.F ? row : g.F - 1) * g.sf + d, VE, t);
#pragma unroll
                for (int e = 0; e < VE; e++) t[e] = there ? t[e] : 0.f;
            } else {
                load_run<TE, VE>(emb + row * g.sf + d, there ? left : 0, t);
            }
        };
        auto multiply = [&](int k, const float (&t)[VE]) {
            const int j = 4 * k + q;
#pragma unroll
            for (int i = 0; i < RT; i++) {
                const float w = j < g.nf ? mine[i][j] : 0.f;            // rows of S behind the last repeat row 0; not stored
#pragma unroll
                for (int e = 0; e < VE; e++) acc[i][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, t[e], acc[i][e], 0, 0, 0);
            }
        };
        float x[VE];
        load_run<T, VE>((const T *)g.x + b * g.ldx + d, g.lead && q == 0 ? left : 0, x);
        auto run = [&](auto fullc) {
            for (int k = 0; k < steps; k += KB) {
                float t[KB][VE];
#pragma unroll
                for (int u = 0; u < KB; u++) rows(k + u, t[u], fullc);
                if (k == 0) {
#pragma unroll
                    for (int e = 0; e < VE; e++) t[0][e] += x[e];       // zero in one of the two
                }
#pragma unroll
                for (int u = 0; u < KB; u++) multiply(k + u, t[u]);
            }
        };
        if (d0 + 16 * VE <= g.D && g.F) run(std::true_type{});
        else run(std::false_type{});
        if (left <= 0) continue;
#pragma unroll
        for (int i = 0; i < RT; i++)
#pragma unroll
            for (int v = 0; v < 4; v++) {
                int row = 16 * i + 4 * q + v;
                if (row >= g.nf) continue;
                float w[VE];
#pragma unroll
                for (int e = 0; e < VE; e++) w[e] = acc[i][e][v];
                if (g.lead) {
                    if (row == 0) {
                        if (g.dx) {
                            float o[VE];
                            load_run<T, VE>(dout + d, left, o);
#pragma unroll
                            for (int e = 0; e < VE; e++) w[e] += o[e];
                            store_run<T, VE>((T *)g.dx + b * g.lddx + d, w, left);
                        }
                        continue;
                    }
                    row--;
                }
                if (g.demb) store_run<TE, VE>((TE *)g.demb + row * g.dsf + b * g.dsb + d, w, left);
            }
    }
}

bool bad(const char *who, const InteractArgs &g, int te, int t) {
    if (g.B < 0 || g.F < 0 || g.D < 0) { set_error("%s: negative size", who); return true; }
    if (te < kF32 || te > kF16 || t < kF32 || t > kF16 || (te != kF32 && te != t)) {
        set_error("%s: type codes %d, %d (embedding rows are float32 or of the output's type)", who, te, t);
        return true;
    }
    if (g.B > ((int64_t)1 << 40)) { set_error("%s: batch of %lld", who, (long long)g.B); return true; }
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

template <class K> int launch(K kernel, const InteractArgs &g, size_t lds, hipStream_t st, int waves = 4) {
    if (lds > 65536) CAFE_HIP_CHECK(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    const int64_t most = (int64_t)1 << 24;                  // samples of a launch: a grid holds fewer than 2^32 work items
    InteractArgs a = g;
    for (a.b0 = 0; a.b0 < g.B; a.b0 += most) {
        const int64_t n = g.B - a.b0 < most ? g.B - a.b0 : most;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((n + waves - 1) / waves)), dim3(64 * waves), lds, st, a);
        CAFE_HIP_CHECK(hipGetLastError());
    }
    return 0;
}
template <class TE, class T> int run_fwd(const InteractArgs &g, hipStream_t st) {
    const size_t lds = (size_t)4 * g.pairs * 4;             // at most 4 waves x 64 * 65 / 2 floats = 33 KB
    if (g.nf <= 16) return launch(k_interact<TE, T, 1>, g, lds, st);
    if (g.nf <= 32) return launch(k_interact<TE, T, 2>, g, lds, st);
    if (g.nf <= 48) return launch(k_interact<TE, T, 3>, g, lds, st);
    if (g.nf <= 64) return launch(k_interact<TE, T, 4>, g, lds, st);
    return launch(k_interact<TE, T, 8>, g, 0, st);
}
template <class TE, class T, int RT> int run_bwd_d(const InteractArgs &g, hipStream_t st) {
    constexpr int W = RT <= 4 ? 4 : 1;                      // S of a wave: at most 64 * 65 floats, 67 KB for four; 128 * 129, 66 KB
    const size_t lds = (size_t)W * g.nf * (g.nf | 1) * 4;
    if (g.D <= 16) return launch(k_interact_bwd<TE, T, RT, 1, W>, g, lds, st, W);
    if (g.D <= 32) return launch(k_interact_bwd<TE, T, RT, 2, W>, g, lds, st, W);
    return launch(k_interact_bwd<TE, T, RT, 4, W>, g, lds, st, W);
}
template <class TE, class T> int run_bwd(const InteractArgs &g, hipStream_t st) {
    if (g.nf <= 16) return run_bwd_d<TE, T, 1>(g, st);
    if (g.nf <= 32) return run_bwd_d<TE, T, 2>(g, st);
    if (g.nf <= 48) return run_bwd_d<TE, T, 3>(g, st);
    if (g.nf <= 64) return run_bwd_d<TE, T, 4>(g, st);
    return run_bwd_d<TE, T, 8>(g, st);
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
