// cafe_adamw.hip -- one AdamW step over many tensors in one launch, moments in float32 or in 8 bits:
//
//     m = b1 m + (1 - b1) g     v = b2 v + (1 - b2) g^2
//     p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// for the dense parameters of the models' heads (the reference steps them with torch.optim).  All arithmetic is float32,
// operation by operation as written (no contraction), so the 8-bit codes do not depend on how a compiler fuses.  Bound by
// memory: 28 bytes per float32 value with float32 moments, 16 with 8-bit ones; 36 M bfloat16 values with 8-bit moments and
// master weights (18 bytes each) take 125-134 us, 4.8-5.2 TB/s, and reading the moments out as float32 (10 bytes) 71.
//
// 8-bit moments.  256 consecutive values share an exponent E, that of the largest finite magnitude among them (at least
// -126; stored plus 127).  A value is scaled by 2^-E -- exactly -- into [0, 2) and rounded in a small floating format: m has a
// sign, 4 exponent and 3 mantissa bits (0x80: not finite, read as NaN), v 5 and 3 (0xff: not finite, read as infinity).  A step
// of the codes is 2^-4 to 2^-3 of a value, over 14 and 30 binades.  The update uses the fresh float32 m and v; only what the
// next step reads is rounded.  A v above 0 is never stored as 0: next step's division by sqrt(v) would blow its m up.
//
// How it is rounded.  One step changes v by some 1 - b2 of itself, a hundredth of a code step, and m by 1 - b1: rounded to
// nearest, they stand still (a constant gradient leaves v at 0.014 of its value after 3000 steps and the parameters go five
// times as far).  So a run of steps rounds up with the probability that the value has of the step above it: the moments are
// then right on average, and noisy by a fifth of v at b2 = 0.999 (3000 steps of constant, random and shrinking gradients: mean
// v 0.99 - 1.01 of the float32 one, parameters within 4 %).  The random bits are a hash of the step's number and the value's
// index: runs repeat, and how tensors are grouped into calls changes nothing.  Nor may a magnitude be cut off at the largest
// code's, 1.75 for v: a block whose largest is above that takes the next exponent.  The first kNearest steps round to nearest
// all the same: the new gradient has a weight of 1 / 8 or more in them, so that moments do not stand still, and nearest is the
// smaller error.  Callers of a single step (dither 0) get nearest, with magnitudes cut off at the largest code.  The hash and
// the registers it holds cost 36 M bfloat16 values with masters 136 us instead of 121, 20 M 68 instead of 64.
#include "cafe_dense.h"

#include <algorithm>
#include <math.h>

using namespace cafe;

namespace {

constexpr int kItems = 48;              // tensors of one launch: their descriptors travel as kernel arguments (4 KB at most)
// Neighbouring values per lane.  8-bit states: 8, so that codes are 8-byte accesses and 32 lanes hold a block (37 M bfloat16
// values with master weights: 138 us; with 4 per lane 149).  float32 states: 4, 16 bytes of each array (200 us; with 8,
// 32 bytes apart, 216).  A workgroup takes 256 times that, without a loop: enough of them are resident to hide the way
// from memory to memory.
constexpr int lane_values(int bits) { return bits == 8 ? 8 : 4; }
constexpr int span(int bits) { return 256 * lane_values(bits); }
constexpr int kBlock = 256;
constexpr int64_t kNearest = 8;         // first steps of a run, whose moments are rounded to nearest
constexpr int64_t kGrid = 1 << 22;      // workgroups of a launch (a grid holds fewer than 2^32 work items); longer tensors go in pieces

struct Item { void *p; const void *g; void *m, *v; uint8_t *me, *ve; float *w; int64_t n; };
struct AdamArgs {
    Item t[kItems];
    int32_t first[kItems + 1];          // first workgroup of every tensor
    const float *factors;               // device: {lr / (1 - b1^t), 1 / sqrt(1 - b2^t), 1 - lr wd}, or null
    float step_size, root, keep, b1, c1, b2, c2, eps;
    int count;
    const int64_t *dither_dev;          // device: the number of the step, or null
    int64_t dither, from;               // the number of the step; values of the first tensor that earlier launches took
};
static_assert(sizeof(AdamArgs) <= 4096, "kernel arguments");

// L elements, at element alignment, as float or int; from `n` on nothing is touched and zeros are read
template <class T, int L> struct __attribute__((packed, aligned(sizeof(T)))) Lane { T e[L]; };
// Past the caches (PAST): what is read or written so is not kept there.
typedef uint32_t past4 __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t past2 __attribute__((ext_vector_type(2), aligned(1)));
template <bool PAST, class U> __device__ __forceinline__ U load_lane(const U *p) {
    if constexpr (!PAST) return *p;
    else if constexpr (sizeof(U) == 8) return __builtin_bit_cast(U, __builtin_nontemporal_load((const past2 *)p));
    else {
        static_assert(sizeof(U) % 16 == 0, "");
        union { U u; past4 v[sizeof(U) / 16]; } x;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(U) / 16); i++) x.v[i] = __builtin_nontemporal_load((const past4 *)p + i);
        return x.u;
    }
}
template <bool PAST, class U> __device__ __forceinline__ void store_lane(U *p, U u) {
    if constexpr (!PAST) *p = u;
    else if constexpr (sizeof(U) == 8) __builtin_nontemporal_store(__builtin_bit_cast(past2, u), (past2 *)p);
    else {
        static_assert(sizeof(U) % 16 == 0, "");
        union { U u; past4 v[sizeof(U) / 16]; } x;
        x.u = u;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(U) / 16); i++) __builtin_nontemporal_store(x.v[i], (past4 *)p + i);
    }
}
template <int L, bool PAST, class T, class F> __device__ __forceinline__ void get(const T *p, int n, F *out) {
    if (n >= L) {
        const Lane<T, L> u = load_lane<PAST>((const Lane<T, L> *)p);
#pragma unroll
        for (int i = 0; i < L; i++) out[i] = (F)u.e[i];
    } else {
#pragma unroll
        for (int i = 0; i < L; i++) out[i] = i < n ? (F)p[i] : (F)0;
    }
}
template <int L, bool PAST, class T, class F> __device__ __forceinline__ void put(T *p, int n, const F *in) {
    Lane<T, L> u;
#pragma unroll
    for (int i = 0; i < L; i++) u.e[i] = (T)in[i];
    if (n >= L) store_lane<PAST>((Lane<T, L> *)p, u);
    else {
#pragma unroll
        for (int i = 0; i < L; i++)
            if (i < n) p[i] = u.e[i];
    }
}

// exponent of |x| with that of 0 and of subnormals taken as -127 (callers clamp)
__device__ __forceinline__ int exponent_of(float mag) { return (int)(__float_as_uint(mag) >> 23) - 127; }

template <bool SECOND> __device__ __forceinline__ float decode8(int c, int e) {
    constexpr int low = SECOND ? -30 : -14;
    const int mag = SECOND ? c : c & 0x7f, field = mag >> 3;
    const float v = ldexpf((float)(field ? 8 + (mag & 7) : mag & 7), (field ? field - 1 : 0) + low - 3 + e);
    if (SECOND) return c == 0xff ? INFINITY : v;
    return c == 0x80 ? NAN : c & 0x80 ? -v : v;
}
// 32 bits that look random, of a counter: two rounds of multiplying by an odd number and folding the high half back (the
// numbers are fractions of the golden ratio and of the square roots of 2 and 3).
constexpr uint32_t kGolden = 0x9E3779B9u;
__device__ __forceinline__ uint32_t scramble(uint32_t h) {
    h ^= h >> 16; h *= 0x6A09E667u;
    h ^= h >> 15; h *= 0xBB67AE85u;
    return h ^ (h >> 16);
}
__device__ __forceinline__ uint32_t dither_key(int64_t step, int64_t index) {
    return scramble(scramble((uint32_t)step * kGolden + (uint32_t)(step >> 32)) + (uint32_t)(index >> 32));
}
// up: in [0, 1), what is added ahead of rounding down; negative: round to nearest even
template <bool SECOND> __device__ __forceinline__ int encode8(float x, int e, float up) {
    constexpr int low = SECOND ? -30 : -14;
    const float mag = fabsf(x);
    if (!(mag <= 3.4028234663852886e38f)) return SECOND ? 0xff : 0x80;
    const float a = ldexpf(mag, -e);
    const int b = max(exponent_of(a), low);
    const float steps = ldexpf(a, 3 - b);
    int c = (int)(up < 0.f ? rintf(steps) : floorf(steps + up)) + 8 * (b - low);
    if (SECOND) {
        c = min(c, 0xfe);
        return c == 0 && mag > 0.f ? 1 : c;
    }
    c = min(c, 0x7f);
    return x < 0.f && c > 0 ? c | 0x80 : c;
}
// Exponents of a block of m and of v, eight values per lane of 32 lanes.  The largest magnitude has the largest exponent and
// leading 7 mantissa bits, so both go through the lanes as the two halves of one word (what is not finite counts as 0).
// ROOM: a block whose largest reaches the largest code takes the next exponent, so that it can be rounded up.
template <bool ROOM> __device__ __forceinline__ void block_exponents(const float *m, const float *v, int *em, int *ev) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t a = (__float_as_uint(m[i]) >> 16) & 0x7fff, b = (__float_as_uint(v[i]) >> 16) & 0x7fff;
        top = __builtin_elementwise_max(top, u16x2{(unsigned short)(a >= 0x7f80 ? 0 : a), (unsigned short)(b >= 0x7f80 ? 0 : b)});
    }
#pragma unroll
    for (int d = 16; d; d >>= 1)
        top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, __shfl_xor(__builtin_bit_cast(int, top), d, 64)));
    *em = max((top.x >> 7) - 127, -126);
    *ev = max((top.y >> 7) - 127, -126);
    if (ROOM) {                                         // 1.875 and 1.75 of that exponent; a byte holds no more than 127
        *em = min(*em + ((top.x & 127) >= 0x70), 127);
        *ev = min(*ev + ((top.y & 127) >= 0x60), 127);
    }
}

__device__ __forceinline__ int item_of(const int32_t *first, int count, int block) {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first[mid] <= block) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// PAST: a step over more than the caches hold.  Nothing of it is found there by the next step, so moments, masters and
// gradients go past them and leave the room to the parameters, which the next forward reads.
// DITHER: 8-bit moments of a run of steps.
template <class T, bool BITS8, bool PAST, bool DITHER> __global__ __launch_bounds__(256) void k_adamw(AdamArgs a) {
    const int k = item_of(a.first, a.count, blockIdx.x);
    const Item t = a.t[k];
    float step_size = a.step_size, root = a.root, keep = a.keep;
    if (a.factors) { step_size = a.factors[0]; root = a.factors[1]; keep = a.factors[2]; }
    constexpr int BITS = BITS8 ? 8 : 32, L = lane_values(BITS);
    const int64_t at = (int64_t)(blockIdx.x - a.first[k]) * span(BITS) + threadIdx.x * L, block = at / kBlock;
    if (block * kBlock >= t.n) return;                  // the block's 32 lanes leave together
    const int n = (int)(t.n - at < L ? t.n - at : L);          // may be <= 0
    float p[L], g[L], m[L], v[L];
    get<L, PAST>((const T *)t.g + at, n, g);
    if (t.w) get<L, PAST>(t.w + at, n, p);
    else get<L, PAST>((const T *)t.p + at, n, p);
    if constexpr (BITS8) {
        int cm[L], cv[L];
        get<L, PAST>((const uint8_t *)t.m + at, n, cm);
        get<L, PAST>((const uint8_t *)t.v + at, n, cv);
        const int em = (int)t.me[block] - 127, ev = (int)t.ve[block] - 127;
#pragma unroll
        for (int i = 0; i < L; i++) { m[i] = decode8<false>(cm[i], em); v[i] = decode8<true>(cv[i], ev); }
    } else {
        get<L, PAST>((const float *)t.m + at, n, m);
        get<L, PAST>((const float *)t.v + at, n, v);
    }
#pragma unroll
    for (int i = 0; i < L; i++) {
        m[i] = m[i] * a.b1 + g[i] * a.c1;
        v[i] = v[i] * a.b2 + (g[i] * g[i]) * a.c2;
        const float denom = sqrtf(v[i]) * root + a.eps;
        p[i] = p[i] * keep - (m[i] / denom) * step_size;
    }
    if constexpr (BITS8) {
#pragma unroll
        for (int i = 0; i < L; i++)
            if (i >= n) m[i] = v[i] = 0.f;
        int em, ev, cm[L], cv[L];
        int64_t run = 0;
        if constexpr (DITHER) run = a.dither_dev ? *a.dither_dev : a.dither;
        if (DITHER && run > kNearest) {
            block_exponents<true>(m, v, &em, &ev);
            const int64_t index = at + (k == 0 ? a.from : 0);
            const uint32_t key = dither_key(run, index);
#pragma unroll
            for (int i = 0; i < L; i++) {               // 20 bits each: steps below 16 and they add up exactly
                const uint32_t h = scramble(((uint32_t)index + i) * kGolden + key);
                cm[i] = encode8<false>(m[i], em, (float)((h << 16 | h >> 16) >> 12) * 0x1p-20f);
                cv[i] = encode8<true>(v[i], ev, (float)(h >> 12) * 0x1p-20f);
            }
        } else {
            block_exponents<false>(m, v, &em, &ev);
#pragma unroll
            for (int i = 0; i < L; i++) { cm[i] = encode8<false>(m[i], em, -1.f); cv[i] = encode8<true>(v[i], ev, -1.f); }
        }
        put<L, PAST>((uint8_t *)t.m + at, n, cm);
        put<L, PAST>((uint8_t *)t.v + at, n, cv);
        if ((threadIdx.x & 31) == 0) { t.me[block] = (uint8_t)(em + 127); t.ve[block] = (uint8_t)(ev + 127); }
    } else {
        put<L, PAST>((float *)t.m + at, n, m);
        put<L, PAST>((float *)t.v + at, n, v);
    }
    if (t.w) put<L, PAST>(t.w + at, n, p);
    put<L, false>((T *)t.p + at, n, p);
}

struct ValueItem { const uint8_t *codes, *exps; float *out; int64_t n; };
struct ValueArgs {
    ValueItem t[2 * kItems];
    int32_t first[2 * kItems + 1];
    uint8_t second[2 * kItems];
    int count;
};
static_assert(sizeof(ValueArgs) <= 4096, "kernel arguments");

template <bool PAST> __global__ __launch_bounds__(256) void k_moment_values(ValueArgs a) {
    const int k = item_of(a.first, a.count, blockIdx.x);
    const ValueItem t = a.t[k];
    const bool second = a.second[k];
    constexpr int L = lane_values(8);
    const int64_t at = (int64_t)(blockIdx.x - a.first[k]) * span(8) + threadIdx.x * L;
    if (at >= t.n) return;
    const int n = (int)(t.n - at < L ? t.n - at : L), e = (int)t.exps[at / kBlock] - 127;
    int c[L];
    float v[L];
    get<L, PAST>(t.codes + at, n, c);
#pragma unroll
    for (int i = 0; i < L; i++) v[i] = second ? decode8<true>(c[i], e) : decode8<false>(c[i], e);
    put<L, PAST>(t.out + at, n, v);
}

__global__ void k_adamw_tick(int64_t *step, const float *lr_dev, double lr, double b1, double b2, double wd, float *factors) {
    const int64_t t = *step + 1;
    *step = t;
    if (lr_dev) lr = (double)*lr_dev;
    factors[0] = (float)(lr / (1.0 - pow(b1, (double)t)));
    factors[1] = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
    factors[2] = (float)(1.0 - lr * wd);
}

bool bad_hyper(const char *who, double lr, double b1, double b2, double eps, double wd) {
    if (!(lr >= 0) || !(b1 >= 0 && b1 < 1) || !(b2 >= 0 && b2 < 1) || !(eps >= 0) || !(wd >= 0)) {
        set_error("%s: lr, eps and weight decay must not be negative, betas lie in [0, 1)", who);
        return true;
    }
    return false;
}

// Bytes of a call from which its arrays go past the caches (256 MB behind the L2s).  A step, with gradients just written
// and parameters read afterwards: 19 M float32 values with float32 moments (528 MB) 133 us, 146 through the caches, 29 M
// 218 and 247, 38 M bfloat16 ones with 8-bit moments and masters (680 MB) 201 and 230; below, 15 M float32 values (411 MB)
// take 115 and 95, 25 M bfloat16 ones (453 MB) 160 and 138.  Reading 38 M moments out twice (302 MB): 71 and 92 us.
constexpr int64_t kPastStep = (int64_t)480 << 20, kPastValues = (int64_t)256 << 20;

template <class T, bool BITS8, bool DITHER> int launch(const AdamArgs &a, unsigned blocks, bool past, hipStream_t st) {
    if (past) hipLaunchKernelGGL((k_adamw<T, BITS8, true, DITHER>), dim3(blocks), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_adamw<T, BITS8, false, DITHER>), dim3(blocks), dim3(256), 0, st, a);
    CAFE_HIP_CHECK(hipGetLastError());
    return 0;
}
template <class T> int launch(const AdamArgs &a, unsigned blocks, bool past, bool eight, hipStream_t st) {
    if (!eight) return launch<T, false, false>(a, blocks, past, st);
    if (a.dither_dev || a.dither > kNearest) return launch<T, true, true>(a, blocks, past, st);
    return launch<T, true, false>(a, blocks, past, st);
}

}  // namespace

extern "C" int cafe_adamw_dev(const int64_t *tensors, int count, int dtype, int state_bits, double lr, double beta1, double beta2,
                              double eps, double weight_decay, int64_t step, const float *d_factors, cafe_stream_t stream) {
    return cafe_adamw_dither_dev(tensors, count, dtype, state_bits, lr, beta1, beta2, eps, weight_decay, step, d_factors, 0, nullptr, stream);
}

extern "C" int cafe_adamw_dither_dev(const int64_t *tensors, int count, int dtype, int state_bits, double lr, double beta1, double beta2,
                                     double eps, double weight_decay, int64_t step, const float *d_factors, int64_t dither,
                                     const int64_t *d_dither, cafe_stream_t stream) {
    if (count < 0 || (count && !tensors)) { set_error("cafe_adamw_dev: no tensor table"); return 1; }
    if (dtype < kF32 || dtype > kF16 || (state_bits != 8 && state_bits != 32)) {
        set_error("cafe_adamw_dev: type code %d, %d-bit states", dtype, state_bits);
        return 1;
    }
    if (bad_hyper("cafe_adamw_dev", lr, beta1, beta2, eps, weight_decay)) return 1;
    if (dither < 0) { set_error("cafe_adamw_dev: dither %lld, 0 or the number of the step expected", (long long)dither); return 1; }
    if (!d_factors && step < 1) { set_error("cafe_adamw_dev: step %lld, the first is 1", (long long)step); return 1; }
    for (int i = 0; i < count; i++) {
        const int64_t *c = tensors + i;
        const int64_t n = c[7 * (int64_t)count];
        bool null = false;
        for (int f = 0; f < 4; f++) null |= c[f * (int64_t)count] == 0;
        if (state_bits == 8) null |= c[4 * (int64_t)count] == 0 || c[5 * (int64_t)count] == 0;
        if (n < 0 || n > ((int64_t)1 << 42) || (n > 0 && null)) {
            set_error("cafe_adamw_dev: tensor %d has %lld values or a null pointer", i, (long long)n);
            return 1;
        }
    }
    AdamArgs a = {};
    a.factors = d_factors;
    a.dither = dither; a.dither_dev = d_dither;
    if (!d_factors) {
        a.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
        a.root = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
        a.keep = (float)(1.0 - lr * weight_decay);
    }
    a.b1 = (float)beta1; a.c1 = (float)(1.0 - beta1); a.b2 = (float)beta2; a.c2 = (float)(1.0 - beta2); a.eps = (float)eps;
    const hipStream_t st = (hipStream_t)stream;
    int64_t bytes = 0;
    for (int k = 0; k < count; k++)
        bytes += tensors[7 * (int64_t)count + k] * ((dtype == kF32 ? 4 : 2) * (tensors[6 * (int64_t)count + k] ? 2 : 3) +
                                                    (tensors[6 * (int64_t)count + k] ? 8 : 0) + (state_bits == 8 ? 4 : 16));
    const bool past = bytes > kPastStep;
    int i = 0;
    int64_t from = 0;                   // values of tensor i that are behind us
    while (i < count) {
        int64_t blocks = 0;
        a.count = 0;
        while (i < count && a.count < kItems && blocks < kGrid) {
            auto at = [&](int f) { return (uintptr_t)tensors[f * (int64_t)count + i]; };
            auto on = [&](int f, int64_t bytes) { return at(f) ? (void *)(at(f) + bytes) : nullptr; };
            const int64_t left = tensors[7 * (int64_t)count + i] - from, n = std::min<int64_t>(left, (kGrid - blocks) * span(state_bits));
            if (left == 0) { i++; from = 0; continue; }
            if (a.count == 0) a.from = from;
            const int64_t e = from * (dtype == kF32 ? 4 : 2), s = state_bits == 8 ? from : from * 4;
            a.t[a.count] = Item{on(0, e), on(1, e), on(2, s), on(3, s), (uint8_t *)on(4, from / kBlock), (uint8_t *)on(5, from / kBlock),
                                (float *)on(6, from * 4), n};
            a.first[a.count++] = (int32_t)blocks;
            blocks += (n + span(state_bits) - 1) / span(state_bits);
            from += n;
        }
        if (!a.count) break;
        a.first[a.count] = (int32_t)blocks;
        const unsigned b = (unsigned)blocks;
        const bool s8 = state_bits == 8;
        const int rc = dtype == kF32 ? launch<float>(a, b, past, s8, st) : dtype == kBF16 ? launch<__bf16>(a, b, past, s8, st)
                                                                                       : launch<_Float16>(a, b, past, s8, st);
        if (rc) return rc;
    }
    return 0;
}

extern "C" int cafe_adamw_tick_dev(int64_t *d_step, const float *d_lr, double lr, double beta1, double beta2, double weight_decay,
                                   float *d_factors, cafe_stream_t stream) {
    if (!d_step || !d_factors) { set_error("cafe_adamw_tick_dev: null pointer"); return 1; }
    if (bad_hyper("cafe_adamw_tick_dev", lr, beta1, beta2, 0, weight_decay)) return 1;
    hipLaunchKernelGGL(k_adamw_tick, dim3(1), dim3(1), 0, (hipStream_t)stream, d_step, d_lr, lr, beta1, beta2, weight_decay, d_factors);
    CAFE_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int cafe_moment8_values_dev(const int64_t *tensors, int count, cafe_stream_t stream) {
    if (count < 0 || (count && !tensors)) { set_error("cafe_moment8_values_dev: no tensor table"); return 1; }
    for (int i = 0; i < count; i++) {
        const int64_t n = tensors[3 * (int64_t)count + i];
        bool null = false;
        for (int f = 0; f < 3; f++) null |= tensors[f * (int64_t)count + i] == 0;
        if (n < 0 || n > ((int64_t)1 << 42) || (n > 0 && null)) {
            set_error("cafe_moment8_values_dev: tensor %d has %lld values or a null pointer", i, (long long)n);
            return 1;
        }
    }
    int64_t bytes = 0;
    for (int k = 0; k < count; k++) bytes += 4 * tensors[3 * (int64_t)count + k];
    const bool past = bytes > kPastValues;
    ValueArgs a = {};
    int i = 0;
    int64_t from = 0;
    while (i < count) {
        int64_t blocks = 0;
        a.count = 0;
        while (i < count && a.count < 2 * kItems && blocks < kGrid) {
            auto at = [&](int f) { return tensors[f * (int64_t)count + i]; };
            const int64_t left = at(3) - from, n = std::min<int64_t>(left, (kGrid - blocks) * span(8));
            if (left == 0) { i++; from = 0; continue; }
            a.t[a.count] = ValueItem{(const uint8_t *)(uintptr_t)at(0) + from, (const uint8_t *)(uintptr_t)at(1) + from / kBlock,
                                     (float *)(uintptr_t)at(2) + from, n};
            a.second[a.count] = at(4) != 0;
            a.first[a.count++] = (int32_t)blocks;
            blocks += (n + span(8) - 1) / span(8);
            from += n;
        }
        if (!a.count) break;
        a.first[a.count] = (int32_t)blocks;
        if (past) hipLaunchKernelGGL(k_moment_values<true>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
        else hipLaunchKernelGGL(k_moment_values<false>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
        CAFE_HIP_CHECK(hipGetLastError());
    }
    return 0;
}
