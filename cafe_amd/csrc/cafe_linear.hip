// cafe_linear.hip -- the matrix products of the models' heads with everything around them in one pass:
//
//     y = act(x W^T + b) + r          x [M, K], W [N, K], b [N], r and y [M, N]
//     dz = dy * act'(z)   dx = dz W   dW = dz^T x   db = sum over rows of dz        (dr = dy)
//
// Reference heads: dlrm_s_pytorch.py:213-251 (Linear + ReLU / Sigmoid layers), wdl.py:704-721 (the wide part's logit
// added to the deep part's sigmoid).  float32, bfloat16 or float16 operands; every sum is a float32 MFMA accumulator.
//
// All three products are  C[i, j] = sum_r A(i, r) B(j, r); an operand is stored either along r ("rows": x and W in the
// forward, dz in dx) or across it ("columns": W in dx; dz and x in dW).  One tile kernel serves them; see k_tile.
#include "cafe_dense.h"

#include <algorithm>

using namespace cafe;

namespace {

// ACT_SLOPE: backward only, the kept values are act'(z) themselves
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SIGMOID = 2, ACT_GELU = 3, ACT_SILU = 4, ACT_COUNT = 5, ACT_SLOPE = 5 };

// act(z), and act'(z) where SLOPE.  relu is told by the sign alone, so its output serves as z in the backward.
// gelu and silu: products with a factor below float32's range are 0, so that infinities give the limits and not NaN.
template <int ACT, bool SLOPE> __device__ __forceinline__ float activate(float z, float *slope) {
    if (ACT == ACT_RELU) {
        if (SLOPE) *slope = z > 0.f ? 1.f : (z != z ? z : 0.f);
        return z > 0.f ? z : (z != z ? z : 0.f);
    }
    if (ACT == ACT_SIGMOID || ACT == ACT_SILU) {
        const float e = expf(-fabsf(z)), q = 1.f / (1.f + e), small = e * q;      // sigmoid(|z|), sigmoid(-|z|)
        const float s = z > 0.f ? q : small, t = z > 0.f ? small : q;             // sigmoid(z), sigmoid(-z)
        if (ACT == ACT_SIGMOID) {
            if (SLOPE) *slope = q * small;
            return z != z ? z : s;
        }
        if (SLOPE) *slope = small == 0.f ? s : s + z * s * t;
        return s == 0.f ? 0.f : z * s;
    }
    if (ACT == ACT_GELU) {                                                        // z Phi(z), no cancellation in the left tail
        const float phi = 0.5f * erfcf(z * -0.70710678f);
        if (SLOPE) {
            const float d = 0.39894228f * expf(-0.5f * z * z);
            *slope = phi + (d == 0.f ? 0.f : z * d);
        }
        return phi == 0.f ? 0.f : z * phi;
    }
    if (SLOPE) *slope = 1.f;
    return z;
}
// act'(z) from what was kept
template <int ACT> __device__ __forceinline__ float act_slope(float kept) {
    if (ACT == ACT_SLOPE) return kept;
    float s;
    activate<ACT, true>(kept, &s);
    return s;
}

// Where a product's result goes.  part != null: float32 partial sums of one slice of the reduction, joined by k_join.
struct Out {
    void *y; int64_t ldy;
    void *kept; int64_t ldk;          // act'(z), in the output's type (null: not wanted)
    const void *bias;
    const void *res; int64_t ldr;
    float *part;
    int act;
};

struct TileArgs {
    const void *a, *b;
    int64_t lda, ldb;
    int64_t I, J, R;                  // C is [I, J], the reduction runs over R
    int tiles_j, tiles;               // tiles along j, tiles in all
    int slices;                       // slices of the reduction (grid.y)
    Out o;
};

template <class T> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mfma32<__bf16>(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma32<_Float16>(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma32<float>(u32x4 a, u32x4 b, f32x16 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int q = 0; q < 4; q++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[q], y[q], c, 0, 0, 0);
    return c;
}
template <class T> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma16<__bf16>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<_Float16>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<float>(u32x4 a, u32x4 b, f32x4 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int q = 0; q < 4; q++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[q], y[q], c, 0, 0, 0);
    return c;
}

// One operand of a tile: BX entries (rows i or j) times BK = 128 bytes' worth of reduction, in LDS.
//   rows (COLS = false):   LDS [BX][128 B + 16 B].  36 banks from row to row: the eight lanes that a 16-byte read serves
//                          together fall on 32 different banks.
//   columns (COLS = true): LDS [BK][BX + pad], as it lies in memory.  float32 reads one value per lane (the two half
//                          waves are 4 rows apart: pad 8 puts them on different halves of the banks); 16-bit types read
//                          through the transposing LDS read, 4 rows x 16 columns per 16 lanes: the row stride is 16 or
//                          48 banks modulo 64, so the 4 rows fall on different banks.
// A lane's fragment for step s holds the reductions 2s+h (h = lane / 32) chunk of 16 bytes in both layouts.
template <class T, bool COLS, int BX, int THREADS> struct Operand {
    static constexpr int E = Elem<T>::per_chunk;
    static constexpr int BK = 8 * E;
    static constexpr int CPR = COLS ? BX / E : 8;                          // 16-byte chunks per LDS row
    static constexpr int ROWS = COLS ? BK : BX;
    static constexpr int PAD = !COLS ? 16 : sizeof(T) == 4 ? 32 : BX == 32 ? 0 : 64;
    static constexpr int STRIDE = CPR * 16 + PAD;                          // bytes
    static constexpr int BYTES = ROWS * STRIDE;
    static constexpr int N = ROWS * CPR / THREADS;                         // chunks per thread
    static constexpr int STEP = THREADS / CPR;                             // rows between a thread's chunks
    static_assert(ROWS * CPR % THREADS == 0 && THREADS % CPR == 0, "");

    const T *p[N];           // first tile's chunks, clamped into the operand
    int64_t adv;             // elements from one tile to the next
    int shift;               // elements to shift a chunk that was moved back to stay inside its row (columns)
    int cols;                // contiguous extent of the operand (columns: of j; rows: of the reduction)
    int64_t R, X, ld, x0;
    const T *base;
    bool tiny;
    u32x4 reg[N];

    __device__ __forceinline__ void init(const void *src, int64_t ld_, int64_t X_, int64_t R_, int64_t x0_) {
        base = (const T *)src; ld = ld_; X = X_; R = R_; x0 = x0_;
        const int t = threadIdx.x, c = t % CPR, row = t / CPR;
        if (COLS) {
            tiny = X < E;
            int64_t col = x0 + c * E, start = col + E > X ? X - E : col;
            if (tiny) start = 0;
            shift = (int)(col - start > E ? E : col - start);
            adv = BK * ld;
#pragma unroll
            for (int n = 0; n < N; n++) p[n] = base + (int64_t)(row + n * STEP) * ld + start;
        } else {
            tiny = R < E;
            shift = 0;
            adv = BK;
#pragma unroll
            for (int n = 0; n < N; n++) {
                int64_t i = x0 + row + n * STEP;
                if (i >= X) i = X - 1;                                     // rows behind the last one repeat it; never stored
                p[n] = base + i * ld + c * E;
            }
        }
    }
    // Requests tile kt.  `last`: the tile that holds the end of the reduction.  What lies outside the operand reads as 0;
    // nothing outside is touched: a chunk that would cross a row's end is read further back and shifted.
    __device__ __forceinline__ void load(int64_t kt, bool last) {
        const int t = threadIdx.x, c = t % CPR, row = t / CPR;
        if (tiny) {
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int64_t r = row + n * STEP;
                if (COLS) reg[n] = kt * BK + r < R ? load_some(base + (kt * BK + r) * ld + x0 + c * E, (int)(X - x0 - c * E)) : u32x4{0, 0, 0, 0};
                else { const int64_t k = kt * BK + c * E; reg[n] = k < R ? load_some(p[n] + kt * BK, (int)(R - k)) : u32x4{0, 0, 0, 0}; }
            }
        } else if (!last) {
#pragma unroll
            for (int n = 0; n < N; n++) reg[n] = load16(p[n] + kt * adv);
        } else if (COLS) {
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int64_t r = kt * BK + row + n * STEP;
                const int64_t back = r < R ? 0 : (r - (R - 1)) * ld;
                reg[n] = load16(p[n] + kt * adv - back);
            }
#pragma unroll
            for (int n = 0; n < N; n++)
                if (kt * BK + row + n * STEP >= R) reg[n] = u32x4{0, 0, 0, 0};
        } else {
            const int64_t k = kt * BK + c * E;
            const int64_t back = k + E > R ? k + E - R : 0;
#pragma unroll
            for (int n = 0; n < N; n++) reg[n] = load16(p[n] + kt * BK - back);
            if (back) {
#pragma unroll
                for (int n = 0; n < N; n++) reg[n] = shift_down<T>(reg[n], back > E ? E : (int)back);
            }
        }
    }
    __device__ __forceinline__ void store(char *lds) const {
        const int t = threadIdx.x, c = t % CPR, row = t / CPR;
#pragma unroll
        for (int n = 0; n < N; n++) {
            u32x4 v = reg[n];
            if (COLS && shift && !tiny) v = shift_down<T>(v, shift);
            *(u32x4 *)(lds + (row + n * STEP) * STRIDE + c * 16) = v;
        }
    }
    // fragment of the 32 entries from x (within the tile) for step s
    __device__ __forceinline__ static u32x4 frag(const char *lds, int x, int s) {
        const int l = threadIdx.x & 63, h = l >> 5;
        if (!COLS) return *(const u32x4 *)(lds + (x + (l & 31)) * STRIDE + (2 * s + h) * 16);
        if constexpr (sizeof(T) == 4) {
            const char *q = lds + (8 * s + 4 * h) * STRIDE + (x + (l & 31)) * 4;
            return u32x4{*(const uint32_t *)q, *(const uint32_t *)(q + STRIDE), *(const uint32_t *)(q + 2 * STRIDE),
                         *(const uint32_t *)(q + 3 * STRIDE)};
        } else {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4 *lp;
            const char *q = lds + (16 * s + 8 * h + ((l & 15) >> 2)) * STRIDE + (x + 16 * ((l >> 4) & 1) + 4 * (l & 3)) * 2;
            const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)q));
            const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(q + 4 * STRIDE)));
            return u32x4{lo.x, lo.y, hi.x, hi.y};
        }
    }
};

// One result: bias, activation, its slope (kept for the backward), residual.
template <class T, int ACT> __device__ __forceinline__ void finish(const Out &o, int64_t i, int64_t j, float v, float bias) {
    v += bias;
    if (o.kept) {
        float s;
        v = activate<ACT, true>(v, &s);
        ((T *)o.kept)[i * o.ldk + j] = (T)s;
    } else {
        v = activate<ACT, false>(v, nullptr);
    }
    if (o.res) v += (float)((const T *)o.res)[i * o.ldr + j];
    ((T *)o.y)[i * o.ldy + j] = (T)v;
}

// C tile of BM x BN by WM x WN waves, each (BM / WM) x (BN / WN) in 32 x 32 MFMA blocks.
template <class T, bool ACOLS, bool BCOLS, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64) void k_tile(TileArgs g) {
    constexpr int TH = WM * WN * 64, TI = BM / WM / 32, TJ = BN / WN / 32;
    typedef Operand<T, ACOLS, BM, TH> OA;
    typedef Operand<T, BCOLS, BN, TH> OB;
    constexpr int BK = OA::BK;
    __shared__ __align__(16) char lds[OA::BYTES + OB::BYTES];
    char *la = lds, *lb = lds + OA::BYTES;
    const int tile = xcd_tile(blockIdx.x, g.tiles);
    const int64_t i0 = (int64_t)(tile / g.tiles_j) * BM, j0 = (int64_t)(tile % g.tiles_j) * BN;
    const int64_t kts = (g.R + BK - 1) / BK;
    const int64_t k0 = kts * blockIdx.y / g.slices, k1 = kts * (blockIdx.y + 1) / g.slices;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int wi = (wave / WN) * (BM / WM), wj = (wave % WN) * (BN / WN);
    f32x16 acc[TI][TJ];
#pragma unroll
    for (int a = 0; a < TI; a++)
#pragma unroll
        for (int b = 0; b < TJ; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[a][b][e] = 0.f;
    OA A; OB B;
    A.init(g.a, g.lda, g.I, g.R, i0);
    B.init(g.b, g.ldb, g.J, g.R, j0);
    if (k0 < k1) { A.load(k0, k0 == kts - 1); B.load(k0, k0 == kts - 1); }
    for (int64_t kt = k0; kt < k1; kt++) {
        A.store(la); B.store(lb);
        __syncthreads();
        if (kt + 1 < k1) { A.load(kt + 1, kt + 1 == kts - 1); B.load(kt + 1, kt + 1 == kts - 1); }
#pragma unroll
        for (int s = 0; s < 4; s++) {
            u32x4 fa[TI], fb[TJ];
#pragma unroll
            for (int a = 0; a < TI; a++) fa[a] = OA::frag(la, wi + 32 * a, s);
#pragma unroll
            for (int b = 0; b < TJ; b++) fb[b] = OB::frag(lb, wj + 32 * b, s);
#pragma unroll
            for (int a = 0; a < TI; a++)
#pragma unroll
                for (int b = 0; b < TJ; b++) acc[a][b] = mfma32<T>(fa[a], fb[b], acc[a][b]);
        }
        __syncthreads();
    }
    // accumulator element e of lane l: row 8 (e / 4) + 4 (l / 32) + e % 4, column l % 32
    const int lj = lane & 31, li = 4 * (lane >> 5);
    if (g.o.part) {
        float *part = g.o.part + (int64_t)blockIdx.y * g.I * g.J;
#pragma unroll
        for (int a = 0; a < TI; a++)
#pragma unroll
            for (int b = 0; b < TJ; b++) {
                const int64_t j = j0 + wj + 32 * b + lj;
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int64_t i = i0 + wi + 32 * a + 8 * (e >> 2) + li + (e & 3);
                    if (i < g.I && j < g.J) part[i * g.J + j] = acc[a][b][e];
                }
            }
        return;
    }
    auto put = [&](auto actc) {
        constexpr int ACT = decltype(actc)::value;
#pragma unroll
        for (int b = 0; b < TJ; b++) {
            const int64_t j = j0 + wj + 32 * b + lj;
            if (j >= g.J) continue;
            const float bias = g.o.bias ? (float)((const T *)g.o.bias)[j] : 0.f;
#pragma unroll
            for (int a = 0; a < TI; a++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int64_t i = i0 + wi + 32 * a + 8 * (e >> 2) + li + (e & 3);
                    if (i < g.I) finish<T, ACT>(g.o, i, j, acc[a][b][e], bias);
                }
        }
    };
    if (!ACOLS && !BCOLS) {
        switch (g.o.act) {
            case ACT_RELU: put(std::integral_constant<int, ACT_RELU>{}); break;
            case ACT_SIGMOID: put(std::integral_constant<int, ACT_SIGMOID>{}); break;
            case ACT_GELU: put(std::integral_constant<int, ACT_GELU>{}); break;
            case ACT_SILU: put(std::integral_constant<int, ACT_SILU>{}); break;
            default: put(std::integral_constant<int, ACT_NONE>{}); break;
        }
    } else {
        put(std::integral_constant<int, ACT_NONE>{});
    }
}

// Sum of the reduction's slices in their order, then what follows the product.
template <class T, int ACT> __global__ __launch_bounds__(256) void k_join(Out o, int64_t I, int64_t J, int slices) {
    const int64_t n = I * J;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < slices; s++) v += o.part[s * n + q];
        const int64_t i = q / J, j = q - i * J;
        finish<T, ACT>(o, i, j, v, o.bias ? (float)((const T *)o.bias)[j] : 0.f);
    }
}

// dz = dy * act'(kept), and the column sums of dz over this block's rows (float32, from the unrounded products).
// A thread holds one 16-byte chunk of columns; blockDim = lanes_x chunks x 256 / lanes_x rows.
template <class T, int ACT>
__global__ __launch_bounds__(256) void k_dz(const T *dy, int64_t ldy, const T *kept, int64_t ldk, T *dz, int64_t M, int N,
                                           int lanes_x, int64_t rows, float *sums) {
    constexpr int E = Elem<T>::per_chunk;
    __shared__ float red[256 * E];
    const int lx = threadIdx.x % lanes_x, ly = threadIdx.x / lanes_x, ny = 256 / lanes_x;
    const int64_t col = ((int64_t)blockIdx.x * lanes_x + lx) * E;
    const int left = (int)(N - col < E ? N - col : E);
    const int64_t m0 = blockIdx.y * rows, m1 = m0 + rows < M ? m0 + rows : M;
    float s[E];
#pragma unroll
    for (int e = 0; e < E; e++) s[e] = 0.f;
    if (left > 0)
        for (int64_t m = m0 + ly; m < m1; m += ny) {
            float g[E];
            unpack<T>(load_some(dy + m * ldy + col, left), g);
            if (ACT != ACT_NONE) {
                float k[E];
                unpack<T>(load_some(kept + m * ldk + col, left), k);
#pragma unroll
                for (int e = 0; e < E; e++) g[e] *= act_slope<ACT>(k[e]);
                store_some(dz + m * N + col, pack<T>(g), left);
            }
#pragma unroll
            for (int e = 0; e < E; e++) s[e] += g[e];
        }
    if (!sums) return;
#pragma unroll
    for (int e = 0; e < E; e++) red[threadIdx.x * E + e] = s[e];
    __syncthreads();
    for (int w = threadIdx.x; w < lanes_x * E; w += 256) {
        const int64_t c = (int64_t)blockIdx.x * lanes_x * E + w;
        if (c >= N) continue;
        float v = 0.f;
        for (int y = 0; y < ny; y++) v += red[y * lanes_x * E + w];
        sums[blockIdx.y * (int64_t)N + c] = v;
    }
}

// db: the blocks' column sums in their order.  64 columns x 4 runs of blocks per workgroup.
template <class T> __global__ __launch_bounds__(256) void k_db(const float *sums, int blocks, int N, T *db) {
    __shared__ float red[256];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), y = threadIdx.x >> 6;
    float v = 0.f;
    if (c < N)
        for (int b = blocks * y / 4; b < blocks * (y + 1) / 4; b++) v += sums[(int64_t)b * N + c];
    red[threadIdx.x] = v;
    __syncthreads();
    if (y == 0 && c < N) db[c] = (T)(red[threadIdx.x] + red[64 + threadIdx.x] + red[128 + threadIdx.x] + red[192 + threadIdx.x]);
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
int64_t elem_size(int dtype) { return dtype == kF32 ? 4 : 2; }
int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// Tile and slices of a product.
struct Plan { int bm, bn; int64_t tiles_i, tiles_j, tiles; int slices; int64_t ws; };

Plan plan(int64_t I, int64_t J, int64_t R, int dtype) {
    Plan p;
    const int64_t bk = 128 / elem_size(dtype), kts = std::max<int64_t>(1, (R + bk - 1) / bk);
    p.bm = I > 64 ? 128 : 64;
    p.bn = J > 64 ? 128 : 64;
    auto count = [&]() { p.tiles_i = (I + p.bm - 1) / p.bm; p.tiles_j = (J + p.bn - 1) / p.bn; p.tiles = p.tiles_i * p.tiles_j; };
    count();
    if (p.tiles < 256) { p.bm = p.bn = 64; count(); }
    p.slices = 1;
    if (p.tiles > 0 && p.tiles < 256) p.slices = (int)std::max<int64_t>(1, std::min<int64_t>({512 / p.tiles, kts / 4, 64}));
    p.ws = p.slices > 1 ? up256((int64_t)p.slices * I * J * 4) : 0;
    return p;
}

template <class T, bool AC, bool BC> int launch_tile(const Plan &p, TileArgs g, hipStream_t st) {
    const dim3 grid((unsigned)p.tiles, (unsigned)p.slices);
    g.tiles_j = (int)p.tiles_j; g.tiles = (int)p.tiles; g.slices = p.slices;
    if (p.bm == 128 && p.bn == 128) hipLaunchKernelGGL((k_tile<T, AC, BC, 128, 128, 2, 2>), grid, dim3(256), 0, st, g);
    else if (p.bm == 128) hipLaunchKernelGGL((k_tile<T, AC, BC, 128, 64, 2, 2>), grid, dim3(256), 0, st, g);
    else if (p.bn == 128) hipLaunchKernelGGL((k_tile<T, AC, BC, 64, 128, 2, 2>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_tile<T, AC, BC, 64, 64, 2, 2>), grid, dim3(256), 0, st, g);
    CAFE_HIP_CHECK(hipGetLastError());
    return 0;
}

template <class F> void with_act(int act, F f) {
    switch (act) {
        case ACT_RELU: f(std::integral_constant<int, ACT_RELU>{}); break;
        case ACT_SIGMOID: f(std::integral_constant<int, ACT_SIGMOID>{}); break;
        case ACT_GELU: f(std::integral_constant<int, ACT_GELU>{}); break;
        case ACT_SILU: f(std::integral_constant<int, ACT_SILU>{}); break;
        case ACT_SLOPE: f(std::integral_constant<int, ACT_SLOPE>{}); break;
        default: f(std::integral_constant<int, ACT_NONE>{}); break;
    }
}

// C = A B (+ what follows) for operands of type T; `part`: workspace of p.ws bytes.
template <class T, bool AC, bool BC> int product(const Plan &p, TileArgs g, float *part, hipStream_t st) {
    if (g.I == 0 || g.J == 0) return 0;
    const Out out = g.o;
    if (p.slices > 1) g.o.part = part;
    if (launch_tile<T, AC, BC>(p, g, st)) return 1;
    if (p.slices > 1) {
        Out o = out;
        o.part = part;
        const unsigned blocks = (unsigned)std::min<int64_t>((g.I * g.J + 255) / 256, 256 * 16);
        with_act(o.act, [&](auto a) { hipLaunchKernelGGL((k_join<T, decltype(a)::value>), dim3(blocks), dim3(256), 0, st, o, g.I, g.J, p.slices); });
        CAFE_HIP_CHECK(hipGetLastError());
    }
    return 0;
}

struct DzPlan { int lanes_x; int64_t blocks_x, blocks_y, rows; };
DzPlan dz_plan(int64_t M, int64_t N, int dtype) {
    DzPlan d;
    const int64_t chunks = (N + 16 / elem_size(dtype) - 1) / (16 / elem_size(dtype));
    d.lanes_x = 1;
    while (d.lanes_x < 64 && d.lanes_x < chunks) d.lanes_x *= 2;
    d.blocks_x = std::max<int64_t>(1, (chunks + d.lanes_x - 1) / d.lanes_x);
    const int64_t ny = 256 / d.lanes_x;
    const int64_t want = std::max<int64_t>(1, 1024 / d.blocks_x);
    d.rows = std::max<int64_t>(ny, (M + want - 1) / want);
    d.rows = (d.rows + ny - 1) / ny * ny;
    d.blocks_y = std::max<int64_t>(1, (M + d.rows - 1) / d.rows);
    return d;
}

// workspace of the backward: [dz][column sums][partial products, used by dx, then by dW]
struct BwdWs { int64_t dz, sums, part, bytes; };
BwdWs bwd_ws(int64_t M, int64_t K, int64_t N, int dtype, int act) {
    BwdWs w;
    const DzPlan d = dz_plan(M, N, dtype);
    w.dz = 0;
    w.sums = act == ACT_NONE ? 0 : up256(M * N * elem_size(dtype));
    w.part = w.sums + up256(d.blocks_y * N * 4);
    w.bytes = w.part + std::max(plan(M, K, N, dtype).ws, plan(N, K, M, dtype).ws);
    return w;
}

bool bad_sizes(const char *who, int64_t m, int64_t k, int64_t n, int dtype, int act, int acts = ACT_COUNT) {
    const int64_t most = INT32_MAX;
    if (m < 0 || k < 0 || n < 0 || m > most || k > most || n > most) {
        set_error("%s: sizes %lld x %lld x %lld outside 0 .. 2^31 - 1", who, (long long)m, (long long)k, (long long)n);
        return true;
    }
    if (dtype < kF32 || dtype > kF16) { set_error("%s: unknown type code %d", who, dtype); return true; }
    if (act < 0 || act >= acts) { set_error("%s: unknown activation code %d", who, act); return true; }
    return false;
}

template <class T> int fwd(TileArgs g, void *ws, int dtype, hipStream_t st) {
    return product<T, false, false>(plan(g.I, g.J, g.R, dtype), g, (float *)ws, st);
}

template <class T>
int bwd(const T *dy, int64_t lddy, const T *x, int64_t ldx, const T *w, int64_t ldw, const T *kept, int64_t ldk, T *dx, int64_t lddx,
        T *dw, T *db, int64_t M, int64_t K, int64_t N, int dtype, int act, char *ws, hipStream_t st) {
    const BwdWs at = bwd_ws(M, K, N, dtype, act);
    const T *dz = dy;
    int64_t lddz = lddy;
    float *sums = (float *)(ws + at.sums), *part = (float *)(ws + at.part);
    const DzPlan d = dz_plan(M, N, dtype);
    if (N > 0 && (act != ACT_NONE || db)) {
        T *z = act != ACT_NONE ? (T *)(ws + at.dz) : nullptr;
        with_act(act, [&](auto a) {
            hipLaunchKernelGGL((k_dz<T, decltype(a)::value>), dim3((unsigned)d.blocks_x, (unsigned)d.blocks_y), dim3(256), 0, st, dy, lddy,
                               kept, ldk, z, M, (int)N, d.lanes_x, d.rows, db ? sums : nullptr);
        });
        CAFE_HIP_CHECK(hipGetLastError());
        if (z) { dz = z; lddz = N; }
        if (db) {
            hipLaunchKernelGGL(k_db<T>, dim3((unsigned)((N + 63) / 64)), dim3(256), 0, st, sums, (int)d.blocks_y, (int)N, db);
            CAFE_HIP_CHECK(hipGetLastError());
        }
    }
    if (dx) {
        TileArgs g = {dz, w, lddz, ldw, M, K, N, 0, 0, 1, {dx, lddx, nullptr, 0, nullptr, nullptr, 0, nullptr, ACT_NONE}};
        if (product<T, false, true>(plan(M, K, N, dtype), g, part, st)) return 1;
    }
    if (dw) {
        TileArgs g = {dz, x, lddz, ldx, N, K, M, 0, 0, 1, {dw, K, nullptr, 0, nullptr, nullptr, 0, nullptr, ACT_NONE}};
        if (product<T, true, true>(plan(N, K, M, dtype), g, part, st)) return 1;
    }
    return 0;
}

}  // namespace

extern "C" int64_t cafe_linear_fwd_ws(int64_t m, int64_t k, int64_t n, int dtype) {
    if (bad_sizes("cafe_linear_fwd_ws", m, k, n, dtype, 0)) return -1;
    return plan(m, n, k, dtype).ws;
}

extern "C" int64_t cafe_linear_bwd_ws(int64_t m, int64_t k, int64_t n, int dtype, int act) {
    if (bad_sizes("cafe_linear_bwd_ws", m, k, n, dtype, act, ACT_SLOPE + 1)) return -1;
    return bwd_ws(m, k, n, dtype, act).bytes;
}

extern "C" int cafe_linear_fwd_dev(const void *d_x, int64_t ldx, const void *d_w, int64_t ldw, const void *d_bias, const void *d_res,
                                   int64_t ldr, void *d_y, int64_t ldy, void *d_kept, int64_t ldk, int64_t m, int64_t k, int64_t n,
                                   int dtype, int act, void *d_ws, int64_t ws_bytes, cafe_stream_t stream) {
    if (bad_sizes("cafe_linear_fwd_dev", m, k, n, dtype, act)) return 1;
    if (m == 0 || n == 0) return 0;
    if (!d_y || (k > 0 && (!d_x || !d_w))) { set_error("cafe_linear_fwd_dev: null pointer"); return 1; }
    if (ldx < 0 || ldw < 0 || ldr < 0 || ldy < n || (d_kept && ldk < n)) { set_error("cafe_linear_fwd_dev: bad row stride"); return 1; }
    const int64_t need = plan(m, n, k, dtype).ws;
    if (ws_bytes < need || (need && !d_ws)) {
        set_error("cafe_linear_fwd_dev: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
        return 1;
    }
    TileArgs g = {d_x, d_w, ldx, ldw, m, n, k, 0, 0, 1, {d_y, ldy, d_kept, ldk, d_bias, d_res, ldr, nullptr, act}};
    const hipStream_t st = (hipStream_t)stream;
    return dtype == kF32 ? fwd<float>(g, d_ws, dtype, st) : dtype == kBF16 ? fwd<__bf16>(g, d_ws, dtype, st) : fwd<_Float16>(g, d_ws, dtype, st);
}

extern "C" int cafe_linear_bwd_dev(const void *d_dy, int64_t lddy, const void *d_x, int64_t ldx, const void *d_w, int64_t ldw,
                                   const void *d_kept, int64_t ldk, void *d_dx, int64_t lddx, void *d_dw, void *d_db, int64_t m, int64_t k,
                                   int64_t n, int dtype, int act, void *d_ws, int64_t ws_bytes, cafe_stream_t stream) {
    if (bad_sizes("cafe_linear_bwd_dev", m, k, n, dtype, act, ACT_SLOPE + 1)) return 1;
    if (m > 0 && n > 0 && (!d_dy || (act != ACT_NONE && !d_kept))) { set_error("cafe_linear_bwd_dev: null gradient or kept values"); return 1; }
    if ((d_dx && m > 0 && n > 0 && k > 0 && !d_w) || (d_dw && m > 0 && n > 0 && k > 0 && !d_x)) { set_error("cafe_linear_bwd_dev: null operand"); return 1; }
    if (lddy < 0 || ldx < 0 || ldw < 0 || ldk < 0 || (d_dx && lddx < k)) { set_error("cafe_linear_bwd_dev: bad row stride"); return 1; }
    const int64_t need = bwd_ws(m, k, n, dtype, act).bytes;
    if (ws_bytes < need || (need && !d_ws)) {
        set_error("cafe_linear_bwd_dev: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
        return 1;
    }
    const hipStream_t st = (hipStream_t)stream;
#define CAFE_BWD(T) bwd<T>((const T *)d_dy, lddy, (const T *)d_x, ldx, (const T *)d_w, ldw, (const T *)d_kept, ldk, (T *)d_dx, lddx, (T *)d_dw, \
                           (T *)d_db, m, k, n, dtype, act, (char *)d_ws, st)
    return dtype == kF32 ? CAFE_BWD(float) : dtype == kBF16 ? CAFE_BWD(__bf16) : CAFE_BWD(_Float16);
#undef CAFE_BWD
}
