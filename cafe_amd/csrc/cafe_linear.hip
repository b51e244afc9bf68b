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

#include <math.h>

#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

using namespace cafe;

namespace {

// ACT_SLOPE: backward only, the kept values are act'(z) themselves
enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SIGMOID = 2, ACT_GELU = 3, ACT_SILU = 4, ACT_COUNT = 5, ACT_SLOPE = 5 };

// e^x for x <= 0, a few 2^-24 off; 0 where that is below float32's normal range, and for NaN.  x log2(e) is carried in two
// parts: rounded to one, the error would grow with x.
__device__ __forceinline__ float exp_low(float x) {
    x = fmaxf(x, -104.f);
    const float y = x * 1.44269504f, rest = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269504f, -y)), e = __builtin_amdgcn_exp2f(y);
    return fmaf(e, rest * 0.693147181f, e);
}
__device__ __forceinline__ float inverse(float d) {                               // of a finite d > 0, one Newton step
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.f), r, r);
}
// act(z), and act'(z) where SLOPE.  relu is told by the sign alone, so its output serves as z in the backward.
// gelu and silu: products with a factor below float32's range are 0, so that infinities give the limits and not NaN.
template <int ACT, bool SLOPE> __device__ __forceinline__ float activate(float z, float *slope) {
    if (ACT == ACT_RELU) {
        if (SLOPE) *slope = z > 0.f ? 1.f : (z != z ? z : 0.f);
        return z > 0.f ? z : (z != z ? z : 0.f);
    }
    if (ACT == ACT_SIGMOID || ACT == ACT_SILU) {
        const float e = exp_low(-fabsf(z)), q = inverse(1.f + e), small = e * q;  // sigmoid(|z|), sigmoid(-|z|)
        const float s = z > 0.f ? q : small, t = z > 0.f ? small : q;             // sigmoid(z), sigmoid(-z)
        if (ACT == ACT_SIGMOID) {
            if (SLOPE) *slope = z != z ? z : q * small;
            return z != z ? z : s;
        }
        if (SLOPE) *slope = z != z ? z : small == 0.f ? s : s + z * s * t;
        return z != z ? z : s == 0.f ? 0.f : z * s;
    }
    // z Phi(z).  Phi(-a) = e^(-a^2 / 2) P(a), no cancellation in the left tail; the slope needs the same exponential.
    // P = t p(t), t = 1 / (1 + 0.35 a), p of degree 9 fitted to erfcx(a / sqrt 2) / 2 over 0 .. 20 (4e-8 of the value
    // off, 4e-7 in float32; erfcf of a rounded z / sqrt 2 was 1e-5 off in the tail).  a^2 is carried in two parts.  Against
    // erfcf, expf and a full division, 8192 x 1024 x 1024 in bfloat16 with slopes takes 34.6 us, not 39.5 (sigmoid 30.3, not
    // 33.4; without an activation 24.4).
    if (ACT == ACT_GELU) {
        const float a = fminf(fabsf(z), 20.f), h = -0.5f * a * a, rest = fmaf(-0.5f * a, a, -h);
        const float e0 = exp_low(h), e = fmaf(e0, rest, e0), t = inverse(fmaf(0.35f, a, 1.f));
        float p = -0.0014221255f;
        p = fmaf(p, t, -0.0218193084f);
        p = fmaf(p, t, 0.127769545f);
        p = fmaf(p, t, -0.235607043f);
        p = fmaf(p, t, 0.143809199f);
        p = fmaf(p, t, -0.0156490859f);
        p = fmaf(p, t, 0.10321828f);
        p = fmaf(p, t, 0.120258741f);
        p = fmaf(p, t, 0.139818564f);
        p = fmaf(p, t, 0.139623225f);
        const float tail = e * t * p, phi = z > 0.f ? 1.f - tail : tail;
        if (SLOPE) {
            const float d = 0.39894228f * e;
            *slope = z != z ? z : phi + (d == 0.f ? 0.f : z * d);
        }
        return z != z ? z : phi == 0.f ? 0.f : z * phi;
    }
    if (SLOPE) *slope = 1.f;
    return z;
}
// dy * act'(z) from what was kept.  Where nothing passes (relu, a slope of 0), nothing of dy does, not even an infinity.
template <int ACT> __device__ __forceinline__ float through(float dy, float kept) {
    if (ACT == ACT_RELU) return kept > 0.f ? dy : (kept != kept ? kept : 0.f);
    if (ACT == ACT_SLOPE) return kept == 0.f ? 0.f : dy * kept;
    float s;
    activate<ACT, true>(kept, &s);
    return s == 0.f ? 0.f : dy * s;
}

// Where a product's result goes.  part != null: float32 partial sums of one slice of the reduction, joined by k_join.
struct Out {
    void *y; int64_t ldy;
    float *kept; int64_t ldk;         // act'(z), unrounded (null: not wanted)
    const void *bias;
    const void *res; int64_t ldr;
    float *part;
    int act;
};

struct TileArgs {
    const void *a, *b;
    int64_t lda, ldb;
    int64_t low;                      // != 0: A is the sum of two matrices, the second that many elements behind the first
    int64_t I, J, R;                  // C is [I, J], the reduction runs over R
    float *sums; void *sums_out;      // column sums of A: per slice, or (one slice) the result itself; null: not wanted
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
// TI x TJ blocks of one step: 16 bytes of reduction per lane on either side.  float32 takes four products per 16 bytes;
// they go round the accumulators, so that neighbours do not depend on each other.
template <class T, int TI, int TJ> __device__ __forceinline__ void mfma_step(const u32x4 *a, const u32x4 *b, f32x16 (*acc)[TJ]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int i = 0; i < TI; i++)
#pragma unroll
                for (int j = 0; j < TJ; j++)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a[i][q]), __uint_as_float(b[j][q]), acc[i][j], 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < TI; i++)
#pragma unroll
            for (int j = 0; j < TJ; j++) acc[i][j] = mfma32<T>(a[i], b[j], acc[i][j]);
    }
}
// One operand of a tile: BX entries (rows i or j) times BK = 128 bytes' worth of reduction, in LDS.
//   rows (COLS = false):   LDS [BX][128 B + 16 B].  36 banks from row to row: the eight lanes that a 16-byte read serves
//                          together fall on 32 different banks.
//   columns (COLS = true): LDS [BK][BX + 32 B], as it lies in memory.  float32 reads one value per lane (the two half waves
//                          are 4 rows apart, on different halves of the banks); 16-bit types read through the transposing
//                          LDS read, 4 rows x 16 columns per 16 lanes, the rows 8 (or 24, 40) banks apart.
// A lane's fragment for step s holds the reductions 2s+h (h = lane / 32) chunk of 16 bytes in both layouts.
// What lies outside the operand reads as 0; nothing outside is touched: a chunk that would cross a row's end is read
// further back and shifted.
// PARTS 2: the operand is the sum of two matrices, BX / 2 entries of the first and the same of the second, `low` elements on.
template <class T, bool COLS, int PARTS, int BX, int THREADS> struct Operand {
    static constexpr int E = Elem<T>::per_chunk;
    static constexpr int BK = 8 * E;
    static constexpr int CPR = COLS ? BX / E : 8;                          // 16-byte chunks per LDS row
    static constexpr int ROWS = COLS ? BK : BX;
    static constexpr int STRIDE = CPR * 16 + (COLS ? 32 : 16);             // bytes
    static constexpr int BYTES = ROWS * STRIDE;
    static constexpr int N = ROWS * CPR / THREADS;                         // chunks per thread
    static constexpr int STEP = THREADS / CPR;                             // rows between a thread's chunks
    static_assert(ROWS * CPR % THREADS == 0 && THREADS % CPR == 0, "");

    const T *p[N];           // first tile's chunks, clamped into the operand
    int64_t adv;             // elements from one tile to the next
    int shift;               // columns: elements to shift a chunk that was moved back to stay inside its row
    bool tiny;               // a row is shorter than a chunk: element by element
    int64_t R, X, ld, x0;
    const T *base;

    static constexpr int ENTRIES = BX / PARTS;                             // rows i or j of the tile
    static_assert(ENTRIES % E == 0, "");

    __device__ __forceinline__ static int column() { return threadIdx.x % CPR * E % ENTRIES; }      // columns: of the thread's chunk
    __device__ __forceinline__ void init(const void *src, int64_t ld_, int64_t X_, int64_t R_, int64_t x0_, int64_t low = 0) {
        base = (const T *)src; ld = ld_; X = X_; R = R_; x0 = x0_;
        const int t = threadIdx.x, c = t % CPR, row = t / CPR;
        if (COLS) {
            if (PARTS > 1 && c * E >= ENTRIES) base += low;
            tiny = X < E;
            int64_t col = x0 + column(), start = col + E > X ? X - E : col;
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
                const int e = row + n * STEP;
                int64_t i = x0 + e % ENTRIES;
                if (i >= X) i = X - 1;                                     // rows behind the last one repeat it; never stored
                p[n] = base + i * ld + c * E + (PARTS > 1 && e >= ENTRIES ? low : 0);
            }
        }
    }
    __device__ __forceinline__ bool edge() const { return COLS && x0 + ENTRIES > X; }       // columns end inside this tile
    // Requests tile kt, which lies inside the operand.
    __device__ __forceinline__ void load_inner(u32x4 (&reg)[N], int64_t kt) const {
#pragma unroll
        for (int n = 0; n < N; n++) reg[n] = load16(p[n] + kt * adv);
    }
    // Requests tile kt.  `last`: the tile that holds the end of the reduction.
    __device__ __forceinline__ void load(u32x4 (&reg)[N], int64_t kt, bool last) const {
        const int t = threadIdx.x, c = t % CPR, row = t / CPR;
        if (!last && !(COLS && tiny)) {
            load_inner(reg, kt);
        } else if (tiny) {
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int64_t r = row + n * STEP;
                if (COLS) reg[n] = kt * BK + r < R ? load_some(base + (kt * BK + r) * ld + x0 + column(), (int)(X - x0 - column())) : u32x4{0, 0, 0, 0};
                else { const int64_t k = kt * BK + c * E; reg[n] = k < R ? load_some(p[n] + kt * BK, (int)(R - k)) : u32x4{0, 0, 0, 0}; }
            }
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
    __device__ __forceinline__ void align(u32x4 (&reg)[N]) const {
        if (edge() && !tiny) {
#pragma unroll
            for (int n = 0; n < N; n++) reg[n] = shift_down<T>(reg[n], shift);
        }
    }
    __device__ __forceinline__ static void store(const u32x4 (&reg)[N], char *lds) {
        const int t = threadIdx.x, c = t % CPR, row = t / CPR;
#pragma unroll
        for (int n = 0; n < N; n++) *(u32x4 *)(lds + (row + n * STEP) * STRIDE + c * 16) = reg[n];
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

// `left` results of one row from column j: bias, activation, its slope (kept for the backward), residual.
template <class T, int ACT> __device__ __forceinline__ void finish(const Out &o, int64_t i, int64_t j, float *v, const float *bias, int left) {
    constexpr int E = Elem<T>::per_chunk;
    float s[E], r[E];
#pragma unroll
    for (int e = 0; e < E; e++) r[e] = 0.f;
    if (o.res) unpack<T>(load_some((const T *)o.res + i * o.ldr + j, left), r);
    if (o.kept) {
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = activate<ACT, true>(v[e] + bias[e], &s[e]);
#pragma unroll
        for (int h = 0; h < E; h += 4) store_some(o.kept + i * o.ldk + j + h, pack<float>(s + h), left - h);
    } else {
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = activate<ACT, false>(v[e] + bias[e], nullptr);
    }
    if (o.res) {
#pragma unroll
        for (int e = 0; e < E; e++) v[e] += r[e];
    }
    store_some((T *)o.y + i * o.ldy + j, pack<T>(v), left);
}
template <class T> __device__ __forceinline__ void bias_chunk(const Out &o, int64_t j, int left, float *b) {
#pragma unroll
    for (int e = 0; e < Elem<T>::per_chunk; e++) b[e] = 0.f;
    if (o.bias) unpack<T>(load_some((const T *)o.bias + j, left), b);
}

// Order of issue for the scheduler: MF products with R LDS reads, W LDS writes and V memory reads spread between them.  A
// wave issues in order: eight writes in a row hold it until LDS has taken them, while the matrix unit runs dry.
template <int MF, int R, int W, int V, int I> __device__ __forceinline__ void weave_one() {
    constexpr int T = R + W + V, m = (I + 1) * MF / T - I * MF / T;
    if constexpr (m > 0) __builtin_amdgcn_sched_group_barrier(0x8, m, 0);
    __builtin_amdgcn_sched_group_barrier(I < R ? 0x100 : I < R + W ? 0x200 : 0x20, 1, 0);
}
template <int MF, int R, int W, int V, int... I> __device__ __forceinline__ void weave_all(std::integer_sequence<int, I...>) {
    (weave_one<MF, R, W, V, I>(), ...);
}
template <int MF, int R, int W, int V> __device__ __forceinline__ void weave() {
    weave_all<MF, R, W, V>(std::make_integer_sequence<int, R + W + V>{});
}

// C tile of BM x BN by WM x WN waves, each (BM / WM) x (BN / WN) in 32 x 32 MFMA blocks.  Two LDS buffers, one barrier per
// 128 bytes of reduction: a wave that writes buffer k % 2 has passed the barrier behind every read of it.  PF tiles are on
// their way in registers: a float32 tile computes for longer than memory takes to answer (64 products of 64 cycles per
// wave), a 16-bit one (16 of 32) does not.
// Bound by the matrix units where the reduction is long: 8192 x 4096 x 2048 takes 980 us in float32 (140 TF; library 912) and
// 155-170 in bfloat16 with normally distributed operands (library 97-113; with uniform ones 132-143 and 87-90: the card's
// clock follows what they toggle), 8192 x 1024 x 1024 139-145 and 22.5.  There the units are busy 76 % of a float32 launch
// (counters), the rest is filling and storing.  Short reductions are bound by what surrounds the products, filling the pipeline
// and passing the tile through LDS: dx at 16384 x 3341 with a reduction of 256 takes 70 us in bfloat16, 1.6 TB/s of stores (66
// with rows on 16-byte boundaries).
//
// PARTS 2: A is the sum of two matrices (dz's rounded values and what their rounding left).  The tile's BM entries are
// BM / 2 rows of both, so that both meet the same B in LDS, and their products are added on the way out.  16384 x 3341 x 256
// in bfloat16, forward and backward, takes 283 us (with one part 215; with the parts one behind the other along the
// reduction 341, registers spilled).
template <class T, bool ACOLS, bool BCOLS, int PARTS, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, 2) void k_tile(TileArgs g) {
    constexpr int TH = WM * WN * 64, TI = BM / WM / 32, TJ = BN / WN / 32, E = Elem<T>::per_chunk, PF = sizeof(T) == 4 ? 1 : 2;
    typedef Operand<T, ACOLS, PARTS, BM, TH> OA;
    typedef Operand<T, BCOLS, 1, BN, TH> OB;
    constexpr int BK = OA::BK, ROWS = BM / PARTS, STAGE = OA::BYTES + OB::BYTES, CS = BN + 8;
    __shared__ __align__(16) char lds[2 * STAGE > BM * CS * 4 ? 2 * STAGE : BM * CS * 4];
    const int tile = xcd_tile(blockIdx.x, g.tiles);
    const int64_t i0 = (int64_t)(tile / g.tiles_j) * ROWS, j0 = (int64_t)(tile % g.tiles_j) * BN;
    const int64_t kts = (g.R + BK - 1) / BK;
    const int64_t k0 = kts * blockIdx.y / g.slices, k1 = kts * (blockIdx.y + 1) / g.slices;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int wi = wave / WN * (BM / WM), wj = wave % WN * (BN / WN);
    f32x16 acc[TI][TJ];
#pragma unroll
    for (int a = 0; a < TI; a++)
#pragma unroll
        for (int b = 0; b < TJ; b++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[a][b][e] = 0.f;
    OA A;
    OB B;
    A.init(g.a, g.lda, g.I, g.R, i0, g.low);
    B.init(g.b, g.ldb, g.J, g.R, j0);
    u32x4 ra[PF][OA::N], rb[PF][OB::N];
    const bool sums = ACOLS && BCOLS && PARTS == 1 && g.sums && j0 == 0;
    float cs[E];
#pragma unroll
    for (int e = 0; e < E; e++) cs[e] = 0.f;

    auto request = [&](int64_t kt, int u, bool inner) {
        if (inner) {
            A.load_inner(ra[u], kt);
            B.load_inner(rb[u], kt);
        } else {
            const bool last = kt == kts - 1;
            A.load(ra[u], kt, last);
            B.load(rb[u], kt, last);
        }
    };
    // Registers of set u -> LDS buffer of tile kt.
    auto stage = [&](int64_t kt, int u, bool woven, bool sums) {
        char *la = lds + (kt & 1) * STAGE, *lb = la + OA::BYTES;
        if (!woven) { A.align(ra[u]); B.align(rb[u]); }
        if (sums) {
#pragma unroll
            for (int n = 0; n < OA::N; n++) {
                float v[E];
                unpack<T>(ra[u][n], v);
#pragma unroll
                for (int e = 0; e < E; e++) cs[e] += v[e];
            }
        }
        OA::store(ra[u], la);
        OB::store(rb[u], lb);
    };
    u32x4 fa[2][TI], fb[2][TJ];
    auto fetch = [&](int64_t kt, int s, int f) {
        const char *la = lds + (kt & 1) * STAGE, *lb = la + OA::BYTES;
#pragma unroll
        for (int a = 0; a < TI; a++) fa[f][a] = OA::frag(la, wi + 32 * a, s);
#pragma unroll
        for (int b = 0; b < TJ; b++) fb[f][b] = OB::frag(lb, wj + 32 * b, s);
    };
    // Tile kt: its first fragments are in set 0.  The next tile goes to LDS behind step 1, the barrier stands behind step
    // 2, and the next tile's first fragments are fetched before step 3's products: the matrix unit always has a step's
    // worth of work while LDS answers.
    // INNER: every tile it touches lies inside the operands and the slice; WOVEN: nor has a chunk to be shifted, and SUMS
    // says whether columns are summed, so that no branch stands between the products (decided at run time instead, sums
    // cost 8192 x 1024 x 1024 in float32 15 us).
    constexpr int MF = TI * TJ * (sizeof(T) == 4 ? 4 : 1), FR = TI * (ACOLS ? 2 : 1) + TJ * (BCOLS ? 2 : 1), MV = OA::N + OB::N;
    auto body = [&](int64_t kt, int u, auto mode) {
        constexpr bool INNER = decltype(mode)::value > 0, WOVEN = decltype(mode)::value >= 2, SUMS = decltype(mode)::value == 3;
        const int un = (u + 1) % PF;
        fetch(kt, 1, 1);
        if (INNER || kt + 1 < k1) stage(kt + 1, un, WOVEN, WOVEN ? SUMS : sums);
        mfma_step<T, TI, TJ>(fa[0], fb[0], acc);
        if constexpr (WOVEN) weave<MF, FR, MV, 0>();
        __builtin_amdgcn_sched_barrier(0);
        fetch(kt, 2, 0);
        if (INNER || kt + 1 + PF < k1) request(kt + 1 + PF, un, INNER);
        mfma_step<T, TI, TJ>(fa[1], fb[1], acc);
        if constexpr (WOVEN) weave<MF, FR, 0, MV>();
        __builtin_amdgcn_sched_barrier(0);
        fetch(kt, 3, 1);
        mfma_step<T, TI, TJ>(fa[0], fb[0], acc);
        if constexpr (WOVEN) weave<MF, FR, 0, 0>();
        __syncthreads();
        if (INNER || kt + 1 < k1) fetch(kt + 1, 0, 0);
        mfma_step<T, TI, TJ>(fa[1], fb[1], acc);
    };
    if (k0 < k1) {
        const bool woven = !(A.edge() || B.edge());
        // tiles that the inner bodies may request: all but the reduction's last, none where rows are shorter than a chunk
        const int64_t inner = A.tiny || B.tiny ? k0 : k1 < kts ? k1 : kts - 1;
        int64_t kt = k0;
        auto start = [&](auto mode) {
            constexpr bool IN = decltype(mode)::value > 0;
#pragma unroll
            for (int u = 0; u < PF; u++)
                if (IN || k0 + u < k1) {
                    request(k0 + u, u, IN);
                    __builtin_amdgcn_sched_barrier(0);          // in this order: the loop waits for the older set
                }
            stage(k0, 0, decltype(mode)::value >= 2, sums);
            if (IN || k0 + PF < k1) request(k0 + PF, 0, IN);
            __syncthreads();
            fetch(k0, 0, 0);
        };
        auto run = [&](auto mode) {
            start(mode);
            for (; kt + 2 * PF < inner; kt += PF) {
#pragma unroll
                for (int u = 0; u < PF; u++) body(kt + u, u, mode);
            }
        };
        if (k0 + 2 * PF >= inner) start(std::integral_constant<int, 0>{});
        else if (woven && !sums) run(std::integral_constant<int, 2>{});
        else if constexpr (ACOLS && BCOLS && PARTS == 1) {
            constexpr int WITH_SUMS = BM < 256 ? 3 : 1;             // 3 would spill registers in the largest tile
            if (woven) run(std::integral_constant<int, WITH_SUMS>{});
            else run(std::integral_constant<int, 1>{});
        } else if constexpr (BCOLS) run(std::integral_constant<int, 1>{});
        for (; kt < k1; kt += PF) {
#pragma unroll
            for (int u = 0; u < PF; u++)
                if (kt + u < k1) body(kt + u, u, std::integral_constant<int, 0>{});
        }
    }
    __syncthreads();

    // The tile goes through LDS, so that a thread ends up with neighbouring columns of a row: 16-byte accesses to
    // everything that follows.  Accumulator element e of lane l: row 8 (e / 4) + 4 (l / 32) + e % 4, column l % 32.
    float *c = (float *)lds;
    if (sums) {                                 // TH / CPR threads hold partial sums of the same columns
        for (int e = 0; e < E; e++) c[threadIdx.x * E + e] = cs[e];
        __syncthreads();
        if (threadIdx.x < BM && i0 + threadIdx.x < g.I) {
            float v = 0.f;
            for (int q = 0; q < OA::STEP; q++) v += c[q * BM + threadIdx.x];
            if (g.sums_out) ((T *)g.sums_out)[i0 + threadIdx.x] = (T)v;
            else g.sums[blockIdx.y * g.I + i0 + threadIdx.x] = v;
        }
        __syncthreads();
    }
    if (!g.o.part && !g.o.y) return;
#pragma unroll
    for (int a = 0; a < TI; a++)
#pragma unroll
        for (int b = 0; b < TJ; b++)
#pragma unroll
            for (int e = 0; e < 16; e++)
                c[(wi + 32 * a + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * CS + wj + 32 * b + (lane & 31)] = acc[a][b][e];
    __syncthreads();
    constexpr int CH = BN / E, PASS = ROWS * CH / TH;
    static_assert(ROWS * CH % TH == 0, "");
    const int col = threadIdx.x % CH * E;
    const int64_t j = j0 + col;
    const int left = (int)(g.J - j < E ? g.J - j : E);
    if (left <= 0) return;
    if (g.o.part) {
        float *part = g.o.part + (int64_t)blockIdx.y * g.I * g.J;
#pragma unroll 2
        for (int q = 0; q < PASS; q++) {
            const int row = threadIdx.x / CH + q * (TH / CH);
            const int64_t i = i0 + row;
            if (i >= g.I) break;
#pragma unroll
            for (int h = 0; h < E; h += 4) {
                f32x4 v = *(const f32x4 *)(c + row * CS + col + h);
                if constexpr (PARTS > 1) v += *(const f32x4 *)(c + (row + ROWS) * CS + col + h);
                store_some(part + i * g.J + j + h, __builtin_bit_cast(u32x4, v), left - h);
            }
        }
        return;
    }
    float bias[E];
    bias_chunk<T>(g.o, j, left, bias);
    auto put = [&](auto actc) {
#pragma unroll 2
        for (int q = 0; q < PASS; q++) {
            const int row = threadIdx.x / CH + q * (TH / CH);
            const int64_t i = i0 + row;
            if (i >= g.I) break;
            float v[E];
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = PARTS > 1 ? c[row * CS + col + e] + c[(row + ROWS) * CS + col + e] : c[row * CS + col + e];
            finish<T, decltype(actc)::value>(g.o, i, j, v, bias, left);
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

// Sum of the reduction's slices in their order, then what follows the product; the blocks behind `out_blocks` join
// `parts` rows of column sums, 16 columns in 16 runs of rows at a time.  Bound by the way of the partial products: 8 slices
// of 1024 x 1024 take 7.6 us (5 TB/s, they are still in the caches).
template <class T, int ACT>
__global__ __launch_bounds__(256) void k_join(Out o, int64_t I, int64_t J, int slices, int out_blocks, const float *sums, int parts, T *sums_out) {
    constexpr int E = Elem<T>::per_chunk;
    if ((int)blockIdx.x >= out_blocks) {
        __shared__ float run[16][16];
        const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
        for (int64_t i0 = (int64_t)(blockIdx.x - out_blocks) * 16; i0 < I; i0 += (int64_t)(gridDim.x - out_blocks) * 16) {
            const int64_t i = i0 + x;
            float v = 0.f;
            if (i < I) {
#pragma unroll 8
                for (int s = parts * y / 16; s < parts * (y + 1) / 16; s++) v += sums[s * I + i];
            }
            run[y][x] = v;
            __syncthreads();
            if (y == 0 && i < I) {
                v = 0.f;
#pragma unroll
                for (int r = 0; r < 16; r++) v += run[r][x];
                sums_out[i] = (T)v;
            }
            __syncthreads();
        }
        return;
    }
    const int64_t chunks = (J + E - 1) / E, n = I * chunks;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (int64_t)out_blocks * 256) {
        const int64_t i = q / chunks, j = (q - i * chunks) * E;
        const int left = (int)(J - j < E ? J - j : E);
        float v[E], bias[E];
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = 0.f;
        const float *part = o.part + i * J + j;
        constexpr int AHEAD = 32 / E;           // slices on their way at a time; added in their order
        int s = 0;
        for (; s + AHEAD <= slices && left >= E; s += AHEAD) {
            u32x4 w[AHEAD][E / 4];
#pragma unroll
            for (int u = 0; u < AHEAD; u++)
#pragma unroll
                for (int h = 0; h < E / 4; h++) w[u][h] = load16(part + (s + u) * (I * J) + 4 * h);
#pragma unroll
            for (int u = 0; u < AHEAD; u++)
#pragma unroll
                for (int e = 0; e < E; e++) v[e] += __uint_as_float(w[u][e / 4][e % 4]);
        }
        for (; s < slices; s++)
#pragma unroll
            for (int h = 0; h < E / 4; h++) {
                const u32x4 w = load_some(part + s * (I * J) + 4 * h, left - 4 * h);
#pragma unroll
                for (int e = 0; e < 4; e++) v[4 * h + e] += __uint_as_float(w[e]);
            }
        bias_chunk<T>(o, j, left, bias);
        finish<T, ACT>(o, i, j, v, bias, left);
    }
}

// y = act(x W^T + b) + r where one side has at most 64 rows (a few samples, or a layer of a few outputs).  Nothing is
// shared between workgroups but the few rows, and there is too little work to fill tiles: a workgroup takes 16 rows of the
// long side (`many`) against all of the short one (FT groups of 16), its WAVES waves take turns along the reduction, and
// operands go from memory to the matrix unit without LDS: lane l holds 16 bytes of row l % 16, chunk l / 16 of the step's
// four, which is the fragment of a 16 x 16 product.  The waves' sums are added through LDS in their order.
// MANY_W: the long side is W (rows of y are the short side's).
struct SkinnyArgs {
    const void *many, *few;
    int64_t ldm, ldf;
    int64_t M, N, K;                  // of the layer
    Out o;
};

template <class T, int FT, int WAVES, bool MANY_W> __global__ __launch_bounds__(WAVES * 64) void k_skinny(SkinnyArgs g) {
    constexpr int E = Elem<T>::per_chunk, STEP = 4 * E, U = FT <= 2 ? 4 : 2;
    __shared__ float part[WAVES][FT * 4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, q = lane >> 4;
    const int64_t many = MANY_W ? g.N : g.M, few = MANY_W ? g.M : g.N, K = g.K;
    const int64_t i0 = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 16;
    if (i0 >= many) return;
    const T *pa = (const T *)g.many + (i0 + r < many ? i0 + r : many - 1) * g.ldm + q * E;
    const T *pb[FT];
#pragma unroll
    for (int f = 0; f < FT; f++) pb[f] = (const T *)g.few + (16 * f + r < few ? 16 * f + r : few - 1) * g.ldf + q * E;
    f32x4 acc[FT];
#pragma unroll
    for (int f = 0; f < FT; f++) acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t whole = K / STEP;                 // steps that lie inside the rows
    int64_t s = wave;
    for (; s + (U - 1) * WAVES < whole; s += U * WAVES) {
        u32x4 a[U], b[U][FT];
#pragma unroll
        for (int u = 0; u < U; u++) {
            a[u] = load16(pa + (s + u * WAVES) * STEP);
#pragma unroll
            for (int f = 0; f < FT; f++) b[u][f] = load16(pb[f] + (s + u * WAVES) * STEP);
        }
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int f = 0; f < FT; f++) acc[f] = mfma16<T>(a[u], b[u][f], acc[f]);
    }
    for (; s * STEP < K; s += WAVES) {
        const int left = (int)(K - s * STEP - q * E < E ? K - s * STEP - q * E : E);
        const u32x4 a = load_some(pa + s * STEP, left);
        u32x4 b[FT];
#pragma unroll
        for (int f = 0; f < FT; f++) b[f] = load_some(pb[f] + s * STEP, left);
#pragma unroll
        for (int f = 0; f < FT; f++) acc[f] = mfma16<T>(a, b[f], acc[f]);
    }
#pragma unroll
    for (int f = 0; f < FT; f++)
#pragma unroll
        for (int e = 0; e < 4; e++) part[wave][f * 4 + e][lane] = acc[f][e];
    __syncthreads();
    // accumulator element e of lane l: long row 4 (l / 16) + e, short row l % 16 of its group
    auto put = [&](auto actc) {
        constexpr int ACT = decltype(actc)::value;
        for (int t = threadIdx.x; t < 256 * FT; t += WAVES * 64) {
            const int i = MANY_W ? t & 15 : (t >> 4) & 15, j = MANY_W ? t >> 4 : (t & 15) + 16 * (t >> 8);
            if (i0 + i >= many || j >= few) continue;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) v += part[w][(j >> 4) * 4 + (i & 3)][16 * (i >> 2) + (j & 15)];
            const int64_t m = MANY_W ? j : i0 + i, n = MANY_W ? i0 + i : j;
            if (g.o.bias) v += (float)((const T *)g.o.bias)[n];
            float slope;
            v = activate<ACT, true>(v, &slope);
            if (g.o.kept) g.o.kept[m * g.o.ldk + n] = slope;
            if (g.o.res) v += (float)((const T *)g.o.res)[m * g.o.ldr + n];
            ((T *)g.o.y)[m * g.o.ldy + n] = (T)v;
        }
    };
    switch (g.o.act) {
        case ACT_RELU: put(std::integral_constant<int, ACT_RELU>{}); break;
        case ACT_SIGMOID: put(std::integral_constant<int, ACT_SIGMOID>{}); break;
        case ACT_GELU: put(std::integral_constant<int, ACT_GELU>{}); break;
        case ACT_SILU: put(std::integral_constant<int, ACT_SILU>{}); break;
        default: put(std::integral_constant<int, ACT_NONE>{}); break;
    }
}

// Whether dz = dy act'(z) of type T is held as two rounded parts: the rounded value, and what the rounding left, rounded.
// Both products take both parts, so that dx and dW carry one rounding, their own (with one part they were 1.4 times as far
// from the exact gradients as those rounded once).  relu and no activation leave dy's own values, which need no rounding.
template <class T, int ACT> constexpr bool two_parts = sizeof(T) == 2 && ACT != ACT_NONE && ACT != ACT_RELU;

// dz = dy * act'(z), rounded; of two parts: what the rounding left, rounded, `low` values further.  kept: z in the type (relu:
// anything of its sign), or the slopes in float32.  One 16-byte chunk per thread and step.  k_dz_sums: and the column sums of
// the unrounded values over the block's rows, a row of `sums` per blockIdx.y; a block has `lanes` chunks side by side.
// Bound by memory: 8192 x 1024 in float32 takes 15.4 us (6.5 TB/s, cached in part), 16384 x 256 in bfloat16 from float32
// slopes, with both parts and the sums, 13.4 (42 MB, 3.1 TB/s).
template <class T, int ACT> __device__ __forceinline__ void dz_chunk(const T *dy, const void *kept, int64_t at_kept, T *dz, int64_t low, int left, float *g) {
    constexpr int E = Elem<T>::per_chunk;
    float k[E];
    unpack<T>(load_some(dy, left), g);
    if constexpr (ACT == ACT_SLOPE) {
#pragma unroll
        for (int h = 0; h < E; h += 4) unpack<float>(load_some((const float *)kept + at_kept + h, left - h), k + h);
    } else {
        unpack<T>(load_some((const T *)kept + at_kept, left), k);
    }
#pragma unroll
    for (int e = 0; e < E; e++) g[e] = through<ACT>(g[e], k[e]);
    const u32x4 high = pack<T>(g);
    store_some(dz, high, left);
    if constexpr (two_parts<T, ACT>) {
        float h[E];
        unpack<T>(high, h);
#pragma unroll
        for (int e = 0; e < E; e++) h[e] = fabsf(h[e]) < INFINITY ? g[e] - h[e] : 0.f;
        store_some(dz + low, pack<T>(h), left);
    }
}
template <class T, int ACT>
__global__ __launch_bounds__(256) void k_dz(const T *dy, int64_t ldy, const void *kept, int64_t ldk, T *dz, int64_t low, int64_t M, int64_t N) {
    constexpr int E = Elem<T>::per_chunk;
    const int64_t chunks = (N + E - 1) / E, n = M * chunks;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n; q += (int64_t)gridDim.x * 256) {
        const int64_t m = q / chunks, col = (q - m * chunks) * E;
        float g[E];
        dz_chunk<T, ACT>(dy + m * ldy + col, kept, m * ldk + col, dz + m * N + col, low, (int)(N - col < E ? N - col : E), g);
    }
}
template <class T, int ACT>
__global__ __launch_bounds__(256) void k_dz_sums(const T *dy, int64_t ldy, const void *kept, int64_t ldk, T *dz, int64_t low, int64_t M, int64_t N,
                                                int lanes, int64_t rows, float *sums) {
    constexpr int E = Elem<T>::per_chunk;
    __shared__ float red[256 * E];
    const int x = threadIdx.x % lanes, y = threadIdx.x / lanes, ny = 256 / lanes;
    const int64_t col = ((int64_t)blockIdx.x * lanes + x) * E, m1 = (blockIdx.y + 1) * rows < M ? (blockIdx.y + 1) * rows : M;
    const int left = (int)(N - col < E ? N - col : E);
    float s[E];
#pragma unroll
    for (int e = 0; e < E; e++) s[e] = 0.f;
    if (left > 0) {
#pragma unroll 4
        for (int64_t m = blockIdx.y * rows + y; m < m1; m += ny) {
            float g[E];
            dz_chunk<T, ACT>(dy + m * ldy + col, kept, m * ldk + col, dz + m * N + col, low, left, g);
#pragma unroll
            for (int e = 0; e < E; e++) s[e] += g[e];
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) red[threadIdx.x * E + e] = s[e];
    __syncthreads();
    for (int w = threadIdx.x; w < lanes * E; w += 256) {
        const int64_t c = (int64_t)blockIdx.x * lanes * E + w;
        if (c >= N) continue;
        float v = 0.f;
        for (int r = 0; r < ny; r++) v += red[r * lanes * E + w];
        sums[blockIdx.y * N + c] = v;
    }
}

// ------------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------------
int64_t elem_size(int dtype) { return dtype == kF32 ? 4 : 2; }
int64_t up256(int64_t v) { return (v + 255) / 256 * 256; }

// Tile and slices of a product: the smallest estimate of its time, in microseconds,
//
//     steps x max(alone, load x shared) + load x ends + join
//
// steps: 128-byte steps of the reduction per slice; load: workgroups per compute unit; shared, alone: what a step costs
// a compute unit among workgroups that fill it and in one that runs by itself (256 x 128 for 16-bit types, 128 x 128, one
// side 64, 64 x 64); ends: loading the first tile and storing the result; join: the second launch, the way of the partial sums
// out and back (2.5 TB/s) and the slices.  The constants are fitted to 1700 timings of 45 products between 1 x 256 x 8192
// and 16384 x 3341 x 256 in float32 and bfloat16; the choice is within 1.2 % of the fastest on average and 25 % off at
// worst (1 x 256 outputs over 8192 in bfloat16).  Both sides of it, bfloat16: 8192 x 256 outputs over 512 take 8.0 us in
// 64 x 64 tiles, 9.6 in 128 x 128 (half the units idle), 12.6 in 256 x 128; 8192 x 1024 over 1024 (dx) take 33.4, 28.4 and
// 22.9; in float32 256 x 128 gains 2 % there and loses 5 % in slices.  float32: 64 x 256 outputs over 8192 take 14.7 us in
// 32 slices and 22 in 12, 128 x 367 over 367 take 9.6 in 4 and 11.9 in 12.
struct Plan { int bm, bn; int64_t tiles_i, tiles_j, tiles; int slices; int64_t ws; double us; };
struct Cost { double shared[4], alone[4], ends, join, per_slice, launch; };

// parts: of the first operand (2: a tile holds half as many of its rows).
Plan plan(int64_t I, int64_t J, int64_t R, int dtype, int parts = 1) {
    static const Cost f32 = {{0, 1.85, 1.01, 0.54}, {0, 2.25, 1.25, 0.68}, 2.4, 1.8, 0.05, 4.8};
    static const Cost half = {{0.92, 0.665, 0.49, 0.27}, {0.98, 0.665, 0.49, 0.293}, 1.25, 2.5, 0.13, 4.55};
    static const struct { int bm, bn, kind; } tiles[] = {{256, 128, 0}, {128, 128, 1}, {128, 64, 2}, {64, 128, 2}, {64, 64, 3}};
    const Cost &c = dtype == kF32 ? f32 : half;
    const int64_t bk = 128 / elem_size(dtype), kts = (R + bk - 1) / bk;
    Plan best = {};
    for (const auto &t : tiles) {
        if (t.kind == 0 && dtype == kF32) continue;
        const int64_t ti = (I + t.bm / parts - 1) / (t.bm / parts), tj = std::max<int64_t>(1, (J + t.bn - 1) / t.bn);
        for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 64}) {
            if (s > 1 && (ti * tj * s > 2048 || kts < 2 * s)) break;
            const double load = std::ceil((double)ti * tj * s / 256.0), steps = (double)((kts + s - 1) / s);
            double us = c.launch + steps * std::max(c.alone[t.kind], c.shared[t.kind] * load) + c.ends * load * (t.bm * t.bn) / 16384.0;
            if (s > 1) us += c.join + c.per_slice * s + 4e-7 * 4 * s * (double)I * J;
            if (best.bm == 0 || us < best.us) best = Plan{t.bm, t.bn, ti, tj, ti * tj, s, 0, us};
        }
    }
    best.ws = best.slices > 1 ? up256((int64_t)best.slices * I * J * 4) : 0;
    return best;
}

template <class T, bool AC, bool BC, int P> int launch_tile_of(const Plan &p, TileArgs g, hipStream_t st) {
    if (p.tiles > (int64_t)1 << 22) {                       // a grid holds fewer than 2^32 work items; INT32_MAX tiles are far behind it
        set_error("cafe_linear: %lld tiles of %d x %d are more than a launch takes", (long long)p.tiles, p.bm, p.bn);
        return 1;
    }
    const dim3 grid((unsigned)g.tiles, (unsigned)p.slices);
    if constexpr (sizeof(T) == 2) {
        if (p.bm == 256) {
            hipLaunchKernelGGL((k_tile<T, AC, BC, P, 256, 128, 4, 2>), grid, dim3(512), 0, st, g);
            CAFE_HIP_CHECK(hipGetLastError());
            return 0;
        }
    }
    // Eight waves where 16-bit types leave each two 32 x 32 blocks (one, in half tiles): the four products of a step are
    // too short to cover a wave's own waits, a second wave on the unit does (16384 x 3341 x 256 in bfloat16 47.8 us, with
    // four waves 51.3; 8192 x 1024 outputs over 479 across rows 15.9 and 19.6).  float32 with eight waves loses 4-10 % in dx.
    constexpr int W = sizeof(T) == 2 ? 2 : 1;
    if (p.bm == 128 && p.bn == 128) hipLaunchKernelGGL((k_tile<T, AC, BC, P, 128, 128, 2, 2 * W>), grid, dim3(256 * W), 0, st, g);
    else if (p.bm == 128) hipLaunchKernelGGL((k_tile<T, AC, BC, P, 128, 64, 2 * W, 2>), grid, dim3(256 * W), 0, st, g);
    else if (p.bn == 128) hipLaunchKernelGGL((k_tile<T, AC, BC, P, 64, 128, 2, 2 * W>), grid, dim3(256 * W), 0, st, g);
    else hipLaunchKernelGGL((k_tile<T, AC, BC, P, 64, 64, 2, 2>), grid, dim3(256), 0, st, g);
    CAFE_HIP_CHECK(hipGetLastError());
    return 0;
}

template <class T, bool AC, bool BC> int launch_tile(const Plan &p, const TileArgs &g, hipStream_t st) {
    if constexpr (sizeof(T) == 2 && BC) {
        if (g.low) return launch_tile_of<T, AC, BC, 2>(p, g, st);
    }
    return launch_tile_of<T, AC, BC, 1>(p, g, st);
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

// Joins a product's slices and `parts` rows of column sums (either may be missing).
template <class T> int join(int slices, const TileArgs &g, const Out &o, float *part, const float *sums, int parts, T *sums_out, hipStream_t st) {
    constexpr int E = Elem<T>::per_chunk;
    Out j = o;
    j.part = part;
    const int out_blocks = part ? (int)std::min<int64_t>((g.I * ((g.J + E - 1) / E) + 255) / 256, 256 * 16) : 0;
    const int sum_blocks = sums_out ? (int)std::min<int64_t>((g.I + 15) / 16, 1 << 16) : 0;
    with_act(o.act, [&](auto a) {
        hipLaunchKernelGGL((k_join<T, decltype(a)::value>), dim3((unsigned)(out_blocks + sum_blocks)), dim3(256), 0, st, j, g.I, g.J, slices,
                           out_blocks, sums, parts, sums_out);
    });
    CAFE_HIP_CHECK(hipGetLastError());
    return 0;
}

// C = A B^T (+ what follows) for operands of type T; `part`, `sums`: workspace.  sums_out: the sums of A's columns (gradient
// of a bias), or null; they are formed here, or were left in `parts` rows of `sums`.  g.o.y == null: the sums alone.
template <class T, bool AC, bool BC>
int product(const Plan &p, TileArgs g, float *part, float *sums, int parts, T *sums_out, hipStream_t st) {
    if (g.I == 0 || (g.J == 0 && !sums_out)) return 0;
    const bool out = g.o.y != nullptr && g.J > 0;
    if (!out && parts) return join<T>(0, g, g.o, nullptr, sums, parts, sums_out, st);
    if (!out) { g.b = g.a; g.ldb = g.lda; g.J = g.I; g.o.y = nullptr; }      // one column of tiles, whose products nobody reads
    const Out o = g.o;
    g.tiles_j = out ? (int)p.tiles_j : 1;
    g.tiles = (int)p.tiles_i * g.tiles_j;
    g.slices = p.slices;
    g.sums = sums_out && !parts ? sums : nullptr;
    g.sums_out = p.slices == 1 ? sums_out : nullptr;
    if (p.slices > 1 && out) g.o.part = part;
    if (launch_tile<T, AC, BC>(p, g, st)) return 1;
    if (p.slices == 1 && !parts) return 0;
    return join<T>(p.slices, g, o, p.slices > 1 && out ? part : nullptr, sums, parts ? parts : p.slices, sums_out, st);
}

// dz is formed once, ahead of both products.  Formed in their loads instead (dy times the slopes, two operands read in place
// of one) it cost float32 more than it saved: 321 us against 307 at 8192 x 1024 x 1024; 16-bit types would read both once
// per column of tiles.  Where dz is rounded, the pass that forms it adds up the bias gradient from the unrounded values;
// elsewhere dW's tiles add up the columns they read anyway.
struct DzPlan { int lanes, parts; int64_t blocks_x, rows; };
int dz_parts(int dtype, int act) { return dtype != kF32 && act != ACT_NONE && act != ACT_RELU ? 2 : 1; }
DzPlan dz_plan(int64_t M, int64_t N, int dtype, int act) {
    DzPlan d = {};
    if (dz_parts(dtype, act) == 1 || M == 0 || N == 0) return d;
    const int64_t chunks = (N + 7) / 8;
    for (d.lanes = 1; d.lanes < 64 && d.lanes < chunks;) d.lanes *= 2;
    d.blocks_x = (chunks + d.lanes - 1) / d.lanes;
    const int64_t ny = 256 / d.lanes, want = std::max<int64_t>(1, std::min<int64_t>(256, 2048 / d.blocks_x));
    d.rows = std::max<int64_t>(ny, (M + want - 1) / want);
    d.parts = (int)((M + d.rows - 1) / d.rows);
    return d;
}

// workspace of the backward: [dz][column sums of the slices or of dz's blocks][partial products, used by dx, then by dW]
struct BwdWs { int64_t sums, part, bytes; };
BwdWs bwd_ws(int64_t M, int64_t K, int64_t N, int dtype, int act) {
    BwdWs w;
    const int parts = dz_parts(dtype, act);
    const Plan dx = plan(M, K, N, dtype, parts), dw = plan(N, K, M, dtype, parts);
    w.sums = act == ACT_NONE ? 0 : up256(parts * M * N * elem_size(dtype));
    w.part = w.sums + up256((int64_t)std::max(dw.slices, dz_plan(M, N, dtype, act).parts) * N * 4);
    w.bytes = w.part + std::max(dx.ws, dw.ws);
    return w;
}

bool bad_sizes(const char *who, int64_t m, int64_t k, int64_t n, int dtype, int act, int acts = ACT_COUNT) {
    const int64_t most = INT32_MAX;
    if (m < 0 || k < 0 || n < 0 || m > most || k > most || n > most) {
        set_error("%s: sizes %lld x %lld x %lld outside 0 .. 2^31 - 1", who, (long long)m, (long long)k, (long long)n);
        return true;
    }
    const int64_t area = (int64_t)1 << 48;                  // values of a matrix: their bytes, twice and in slices, fit 63 bits
    if (m * n > area || m * k > area || n * k > area) {
        set_error("%s: a matrix of %lld x %lld x %lld has more than 2^48 values", who, (long long)m, (long long)k, (long long)n);
        return true;
    }
    if (dtype < kF32 || dtype > kF16) { set_error("%s: unknown type code %d", who, dtype); return true; }
    if (act < 0 || act >= acts) { set_error("%s: unknown activation code %d", who, act); return true; }
    return false;
}

template <class T, int FT, bool MANY_W> int launch_skinny(const SkinnyArgs &g, hipStream_t st) {
    const int64_t many = MANY_W ? g.N : g.M;
    const int64_t blocks = (many + 15) / 16, wide = 1 << 20;
    const dim3 grid((unsigned)std::min(blocks, wide), (unsigned)((blocks + wide - 1) / wide));
    if (many <= 16 * 512) hipLaunchKernelGGL((k_skinny<T, FT, 8, MANY_W>), grid, dim3(512), 0, st, g);
    else hipLaunchKernelGGL((k_skinny<T, FT, 4, MANY_W>), grid, dim3(256), 0, st, g);
    CAFE_HIP_CHECK(hipGetLastError());
    return 0;
}
template <class T, bool MANY_W> int skinny(const SkinnyArgs &g, hipStream_t st) {
    const int64_t few = MANY_W ? g.M : g.N;
    if (few <= 16) return launch_skinny<T, 1, MANY_W>(g, st);
    if (few <= 32) return launch_skinny<T, 2, MANY_W>(g, st);
    return launch_skinny<T, 4, MANY_W>(g, st);
}
// Estimate of k_skinny's time, in microseconds: the waves' way along a row (a memory latency per batch of loads, dearer with
// every short row; four times that where 16-bit rows start at odd addresses: 1 x 3341 x 1024 in bfloat16 takes 11.9 us,
// 1 x 3344 x 1024 takes 4.6) or the rows' way from memory.  At 1 x 479 x 1024 it takes 4.6 us in bfloat16 (the tiles 6.6),
// at 8192 x 256 x 1 in float32 4.2 (the tiles 9.5), at 64 x 1024 x 1024 in float32 12.8 (the tiles 9.7).
double skinny_us(int64_t m, int64_t k, int64_t n, int dtype, bool aligned) {
    const double few = (double)std::min(m, n), many = (double)std::max(m, n), row = (double)k * elem_size(dtype);
    return 2.9 + std::max(row * (0.0005 + 0.000025 * few) * (aligned ? 1 : 4), many * row * (aligned ? 1 : 2) * (1 + few / 64) / 5e6);
}
bool is_skinny(int64_t m, int64_t k, int64_t n, int dtype, bool aligned) {
    return std::min(m, n) <= 64 && skinny_us(m, k, n, dtype, aligned) < plan(m, n, k, dtype).us;
}

template <class T> int fwd(TileArgs g, void *ws, int dtype, hipStream_t st) {
    const bool aligned = sizeof(T) == 4 || (((g.lda | g.ldb) & 1) == 0 && (((uintptr_t)g.a | (uintptr_t)g.b) & 3) == 0);
    if (is_skinny(g.I, g.R, g.J, dtype, aligned)) {
        if (g.I <= g.J) return skinny<T, true>(SkinnyArgs{g.b, g.a, g.ldb, g.lda, g.I, g.J, g.R, g.o}, st);
        return skinny<T, false>(SkinnyArgs{g.a, g.b, g.lda, g.ldb, g.I, g.J, g.R, g.o}, st);
    }
    return product<T, false, false>(plan(g.I, g.J, g.R, dtype), g, (float *)ws, nullptr, 0, nullptr, st);
}
int64_t fwd_ws(int64_t m, int64_t k, int64_t n, int dtype) {
    return is_skinny(m, k, n, dtype, dtype == kF32) ? 0 : plan(m, n, k, dtype).ws;      // whatever the alignment turns out to be
}

template <class T>
int bwd(const T *dy, int64_t lddy, const T *x, int64_t ldx, const T *w, int64_t ldw, const void *kept, int64_t ldk, T *dx, int64_t lddx,
        T *dw, T *db, int64_t M, int64_t K, int64_t N, int dtype, int act, char *ws, hipStream_t st) {
    const BwdWs at = bwd_ws(M, K, N, dtype, act);
    float *sums = (float *)(ws + at.sums), *part = (float *)(ws + at.part);
    const T *dz = dy;
    int64_t lddz = lddy;
    DzPlan d = {};
    const int parts = dz_parts(dtype, act);
    const int64_t low = parts == 2 ? M * N : 0;
    if (act != ACT_NONE && M > 0 && N > 0 && (dx || dw || db)) {
        T *z = (T *)ws;
        constexpr int E = Elem<T>::per_chunk;
        const unsigned blocks = (unsigned)std::min<int64_t>((M * ((N + E - 1) / E) + 255) / 256, 256 * 32);
        if (db) d = dz_plan(M, N, dtype, act);
        with_act(act, [&](auto a) {
            constexpr int ACT = decltype(a)::value;
            if (d.parts) hipLaunchKernelGGL((k_dz_sums<T, ACT>), dim3((unsigned)d.blocks_x, (unsigned)d.parts), dim3(256), 0, st, dy, lddy, kept,
                                            ldk, z, low, M, N, d.lanes, d.rows, sums);
            else hipLaunchKernelGGL((k_dz<T, ACT>), dim3(blocks), dim3(256), 0, st, dy, lddy, kept, ldk, z, low, M, N);
        });
        CAFE_HIP_CHECK(hipGetLastError());
        dz = z; lddz = N;
    }
    TileArgs g = {};
    g.a = dz; g.lda = lddz; g.low = low;
    if (dx) {
        TileArgs q = g;
        q.b = w; q.ldb = ldw; q.I = M; q.J = K; q.R = N;
        q.o.y = dx; q.o.ldy = lddx;
        if (product<T, false, true>(plan(M, K, N, dtype, parts), q, part, nullptr, 0, nullptr, st)) return 1;
    }
    if (dw || db) {
        TileArgs q = g;
        q.b = x; q.ldb = ldx; q.I = N; q.J = K; q.R = M;
        q.o.y = dw; q.o.ldy = K;
        return product<T, true, true>(plan(N, K, M, dtype, parts), q, part, sums, d.parts, db, st);
    }
    return 0;
}

}  // namespace

extern "C" int64_t cafe_linear_fwd_ws(int64_t m, int64_t k, int64_t n, int dtype) {
    if (bad_sizes("cafe_linear_fwd_ws", m, k, n, dtype, 0)) return -1;
    return fwd_ws(m, k, n, dtype);
}

extern "C" int64_t cafe_linear_bwd_ws(int64_t m, int64_t k, int64_t n, int dtype, int act) {
    if (bad_sizes("cafe_linear_bwd_ws", m, k, n, dtype, act, ACT_SLOPE + 1)) return -1;
    return bwd_ws(m, k, n, dtype, act).bytes;
}

extern "C" int cafe_linear_plan(int64_t m, int64_t k, int64_t n, int dtype, int act, int product, int *tile) {
    if (bad_sizes("cafe_linear_plan", m, k, n, dtype, act, ACT_SLOPE + 1)) return 1;
    if (product < 0 || product > 2 || !tile) { set_error("cafe_linear_plan: product %d, or no array", product); return 1; }
    const int parts = product ? dz_parts(dtype, act) : 1;
    const Plan p = product == 0 ? plan(m, n, k, dtype) : product == 1 ? plan(m, k, n, dtype, parts) : plan(n, k, m, dtype, parts);
    const bool few = product == 0 && is_skinny(m, k, n, dtype, true);
    tile[0] = few ? 0 : p.bm; tile[1] = few ? 0 : p.bn; tile[2] = few ? 1 : p.slices; tile[3] = parts;
    return 0;
}

extern "C" int cafe_linear_fwd_dev(const void *d_x, int64_t ldx, const void *d_w, int64_t ldw, const void *d_bias, const void *d_res,
                                   int64_t ldr, void *d_y, int64_t ldy, float *d_kept, int64_t ldk, int64_t m, int64_t k, int64_t n,
                                   int dtype, int act, void *d_ws, int64_t ws_bytes, cafe_stream_t stream) {
    if (bad_sizes("cafe_linear_fwd_dev", m, k, n, dtype, act)) return 1;
    if (m == 0 || n == 0) return 0;
    if (!d_y || (k > 0 && (!d_x || !d_w))) { set_error("cafe_linear_fwd_dev: null pointer"); return 1; }
    if (ldx < 0 || ldw < 0 || ldr < 0 || ldy < n || (d_kept && ldk < n)) { set_error("cafe_linear_fwd_dev: bad row stride"); return 1; }
    const int64_t need = fwd_ws(m, k, n, dtype);
    if (ws_bytes < need || (need && !d_ws)) {
        set_error("cafe_linear_fwd_dev: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
        return 1;
    }
    TileArgs g = {};
    g.a = d_x; g.lda = ldx; g.b = d_w; g.ldb = ldw; g.I = m; g.J = n; g.R = k;
    g.o = Out{d_y, ldy, d_kept, ldk, d_bias, d_res, ldr, nullptr, act};
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
#define CAFE_BWD(T) bwd<T>((const T *)d_dy, lddy, (const T *)d_x, ldx, (const T *)d_w, ldw, d_kept, ldk, (T *)d_dx, lddx, (T *)d_dw, \
                           (T *)d_db, m, k, n, dtype, act, (char *)d_ws, st)
    return dtype == kF32 ? CAFE_BWD(float) : dtype == kBF16 ? CAFE_BWD(__bf16) : CAFE_BWD(_Float16);
#undef CAFE_BWD
}
