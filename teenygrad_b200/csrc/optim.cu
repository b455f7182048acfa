// The optimiser's side of the training step: the norm of all gradients, and
// AdamW over many tensors in one launch with its moments in 32 bits or in 8
// (the reference's LoadedModel::adamw_step, drivers/teeny-cuda/src/model/mod.rs:868).
//
//   g' = g * grad_scale        m = b1 m + (1 - b1) g'      v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by HBM: every value is read once and written once.  The table of tensors
// rides in the launch's parameters, so a step copies nothing to the device, needs
// no workspace and can be captured; the grid walks the chunks of all tensors with
// its stride, so that small tensors share a wave and large ones are split.
//
// 8-bit moments.  m and s = sqrt(v) are held as e4m3 codes, one power of two a
// block of 256 elements: value = code * 2^(exp - 127), the exponent that puts the
// block's largest value in [128, 256).
//  * A power of two makes the decoding exact and costs a floating code nothing.
//  * s in place of v: its code spans 2^17 below the block's largest, as m's does,
//    where v's would span 2^8.5 of it; and a root above zero is never stored as
//    zero, since p's step divides by it.
//  * b2 = 0.999 moves v by a thousandth a step, which an 8-bit code rounded to
//    nearest never follows.  The codes are rounded up or down with the
//    probability of the rest, by 16 bits each of a hash of (seed, step, tensor,
//    element), and a run repeats.  The mean of m over the steps is the 32-bit
//    moment's.  s has no bias of its own either, but v is its square, high by the
//    rounding's variance: by 4.6 % for normal gradients whatever b2 is, by 10 %
//    where s is 4 to 8 times the smallest code, by more below that, where a root
//    above zero also stays a code above zero.
//  * Each operation up to the code is rounded by itself (no fused multiply-add),
//    so the codes are defined bit for bit by the formula.
//
// Measured over 1e9 parameters, steps back to back (the floor is the bytes at the rate
// of a copy, 6.45 TB/s): f32 moments, f32 parameters and gradients 4.37 ms (floor 4.34),
// bf16 gradients 4.14 (4.03), and a bf16 copy 4.65 (4.34), all bf16 3.56 (3.41); 8-bit
// moments 2.76 (2.48), 2.62 (2.17), 2.81 (2.48) and 2.24 (1.55).  A step by itself, at the
// highest clock, takes 2.47, 2.43, 2.54 and 2.18 ms with 8-bit moments: with f32 parameters
// HBM is the bound there, and instruction issue (56 of them an element) at the clock that
// steps back to back leave; with bf16 parameters issue is in both.  1.1e9 bf16 gradients'
// norm 0.32 ms.
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <float.h>
#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <new>

#include "common.cuh"
#include "f32x2.cuh"

namespace tb {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kBlock = 256;       // elements that share an exponent: one warp, 8 a lane
constexpr int kThreads = 256;
constexpr int kChunk = 2048;      // elements of one tensor that a CTA takes at a time
constexpr int kNormChunk = 8192;  // the same of the gradient norm
constexpr int kCtasPerSm = 4;
constexpr int kUnit8 = 2 * kBlock;                // 8-bit: what a warp takes at a time
constexpr int kThreads8 = 64;
constexpr int kChunk8 = kThreads8 / 32 * kUnit8;

// Tensors a launch's parameters hold.  A call with 4 KB of them takes the host 3.1
// us (48 tensors), with 32 KB 4.9 (49), so models of few tensors take the small table.
constexpr int kSmallTable = 48, kLargeTable = 440;

struct Entry {
    void* p;
    const void* g;
    void* m;
    void* v;
    uint8_t* m_exp;
    uint8_t* v_exp;
    void* copy;
    int64_t n;
};

struct Hyper {
    float lr, beta1, beta2, rest1, rest2, eps, decay, log1, log2;   // rest = 1 - beta, log = log(beta)
    int64_t step;
    const float* lr_dev;
    const float* grad_scale;
    const int64_t* step_dev;
    uint32_t seed;
    uint32_t first;   // number of the table's first tensor
};

template <int CAP>
struct Table {
    Entry e[CAP];
    int start[CAP + 1];   // first chunk of each tensor; the last entry is the number of chunks
    int whole[CAP];       // units of kUnit8 that are whole and at aligned addresses
    uint8_t vec[CAP];     // the tensor's addresses allow vector accesses
    int n;
    Hyper h;
};
static_assert(sizeof(Table<kSmallTable>) <= 4096 - 256, "fits the small parameter space");
static_assert(sizeof(Table<kLargeTable>) <= 32764 - 256, "fits the parameter space");

// The tensor that holds a chunk.
template <int CAP>
__device__ __forceinline__ int find(const Table<CAP>& t, int chunk) {
    int lo = 0, hi = t.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.start[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The same for a chunk at or after one that tensor k holds: the grid's stride passes
// few tensors at a time.
template <int CAP>
__device__ __forceinline__ int advance(const Table<CAP>& t, int k, int chunk) {
    while (t.start[k + 1] <= chunk) k++;
    return k;
}

// ------------------------------------------------------------------ loads --
__device__ __forceinline__ void load4(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
__device__ __forceinline__ void load4(const bf16* p, float* v) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(a.x); v[1] = bf16_hi(a.x); v[2] = bf16_lo(a.y); v[3] = bf16_hi(a.y);
}
__device__ __forceinline__ void store4(float* p, const float* v) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(bf16* p, const float* v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

// Four elements from i of an array of n, zeros past its end.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int64_t i, int64_t n, bool vec, float* v) {
    if (vec && i + 4 <= n) {
        load4(p + i, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++) v[j] = i + j < n ? load1(p + i + j) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int64_t i, int64_t n, bool vec, const float* v) {
    if (vec && i + 4 <= n) {
        store4(p + i, v);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (i + j < n) store1(p + i + j, v[j]);
}
// ------------------------------------------------------------------ AdamW --
// The step's scalars.
struct Step {
    float scale, keep, rate, root, eps;   // keep = 1 - lr wd, rate = lr / (1 - b1^t), root = 1 / sqrt(1 - b2^t)
    // A root that the hardware's flushes to 0 is under 2^-63: times `root`, under 2^-24 of an eps above this.
    float flushed;
    uint32_t key;
};

// Xor-shifts and odd multipliers (the fractions of sqrt 2 and sqrt 3), each a bijection.
__device__ __forceinline__ uint32_t mix_most(uint32_t x) {
    x ^= x >> 16;
    x *= 0x6A09E667u;
    x ^= x >> 15;
    return x * 0xBB67AE85u;
}
__device__ __forceinline__ uint32_t mix(uint32_t x) {
    x = mix_most(x);
    return x ^ (x >> 16);
}

__device__ __forceinline__ Step step_of(const Hyper& h) {
    const int64_t t = h.step_dev ? *h.step_dev : h.step;
    const float lr = h.lr_dev ? *h.lr_dev : h.lr;
    Step s;
    s.scale = h.grad_scale ? *h.grad_scale : 1.f;
    s.keep = 1.f - lr * h.decay;
    // 1 - beta^t = -expm1(t log(beta)): no cancellation at the first steps
    s.rate = lr / -expm1f((float)t * h.log1);
    s.root = rsqrtf(-expm1f((float)t * h.log2));
    s.eps = h.eps;
    s.flushed = fmaxf(0x1p-39f * s.root, 1e-30f);
    s.key = mix(mix(h.seed) ^ (uint32_t)t);
    return s;
}

// The quotient has 2 units in the last place; a numerator under 2^-126 counts as 0.
__device__ __forceinline__ float stepped(float p, float m, float root_v, const Step& s) {
    float q;
    asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(q) : "f"(s.rate * m), "f"(root_v * s.root + s.eps));
    return p * s.keep - q;
}

// CTAs an SM: as many as keep HBM busy, since more of them cost DRAM rows.  1e9 parameters, back to back, with 2 / 3 / 4
// CTAs: f32 and f32 gradients 4.37 / 4.65 / 4.70 ms, bf16 gradients 4.72 / 4.15 / 4.39 and with the copy 5.01 / 4.64 /
// 4.78, bf16 and bf16 4.38 / 3.69 / 3.57.  (The floors are 4.34, 4.03, 4.34 and 3.41.)
template <typename P, typename G>
constexpr int adamw_ctas() {
    return sizeof(P) == 2 ? 4 : sizeof(G) == 2 ? 3 : 2;
}

template <typename P, typename G, int CAP>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) adamw_kernel(const __grid_constant__ Table<CAP> t) {
    const Step s = step_of(t.h);
    const float b1 = t.h.beta1, b2 = t.h.beta2, r1 = t.h.rest1, r2 = t.h.rest2;
    const int chunks = t.start[t.n];
    int k = find(t, blockIdx.x);
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        k = advance(t, k, c);
        const Entry& e = t.e[k];
        const bool vec = t.vec[k];
        const int64_t n = e.n, i0 = (int64_t)(c - t.start[k]) * kChunk + threadIdx.x * 4;
        P* pp = (P*)e.p;
        const G* pg = (const G*)e.g;
        float *pm = (float*)e.m, *pv = (float*)e.v;
        float p[2][4], g[2][4], m[2][4], v[2][4];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int64_t i = i0 + u * (kChunk / 2);
            if (i >= n) continue;
            load4(pp, i, n, vec, p[u]);
            load4(pg, i, n, vec, g[u]);
            load4(pm, i, n, vec, m[u]);
            load4(pv, i, n, vec, v[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int64_t i = i0 + u * (kChunk / 2);
            if (i >= n) continue;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float gj = g[u][j] * s.scale;
                m[u][j] = b1 * m[u][j] + r1 * gj;
                v[u][j] = b2 * v[u][j] + r2 * gj * gj;
                p[u][j] = stepped(p[u][j], m[u][j], sqrtf(v[u][j]), s);
            }
            store4(pp, i, n, vec, p[u]);
            store4(pm, i, n, vec, m[u]);
            store4(pv, i, n, vec, v[u]);
            if (e.copy) store4((bf16*)e.copy, i, n, vec, p[u]);
        }
    }
}

// Two sums.  Packed, they were contracted with the products they add; scalar ones with a rounding of their own are not.
__device__ __forceinline__ void sums(F2 a, F2 b, float* v) {
    float x[2], y[2];
    get(a, x);
    get(b, y);
    v[0] = __fadd_rn(x[0], y[0]);
    v[1] = __fadd_rn(x[1], y[1]);
}
// The largest of three sizes; NaN where one is NaN.
__device__ __forceinline__ float largest(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float sqrt_fast(float x) {
    float y;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ------------------------------------------------------------ 8-bit codes --
// 2^e for e in [-149, 127], exact.
__device__ __forceinline__ float power(int e) {
    return __uint_as_float(e >= -126 ? (uint32_t)(e + 127) << 23 : 1u << (e + 149));
}

__device__ __forceinline__ void decode4(uint32_t w, float* v) {
    const __half2 a(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3));
    const __half2 b(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3));
    const float2 x = __half22float2(a), y = __half22float2(b);
    v[0] = x.x; v[1] = x.y; v[2] = y.x; v[3] = y.y;
}

// The block's exponent for its largest value's bits: that of its binade, less 7.
__device__ __forceinline__ int block_exponent(uint32_t top) { return (int)max(top >> 23, 7u) - 7; }

// Codes.  x is scaled to put the code's smallest normal value, 2^-6, on f32's, 2^-126: then
// the code is the f32's bits 20 to 26, in the subnormal range too, and what lies below them
// carries into it with probability rest / 2^20 when 16 random bits (and a half) are added.
constexpr int kCodeScale = -120;

// 16 random bits and a half each, from bit 8 on: with bits = mix(x), rm = (bits & 0xffff) << 8 | 0x80 and
// rs = bits >> 16 << 8 | 0x80.  mix's last step only changes the low half, by the high one.
__device__ __forceinline__ void random_bits(uint32_t x, uint32_t& rm, uint32_t& rs) {
    x = mix_most(x);
    rs = __byte_perm(x, 0x80u, 0x5324);
    rm = __byte_perm(x, 0u, 0x4104) ^ rs;
}

// Bytes 3 of four words.
__device__ __forceinline__ uint32_t top_bytes(const uint32_t* t) {
    return __byte_perm(__byte_perm(t[0], t[1], 0x0073), __byte_perm(t[2], t[3], 0x7300), 0x7610);
}

// The code of a value of any kind: what is not finite becomes NaN; the scaling in two steps.
__device__ __forceinline__ uint32_t any_code(float x, int e, uint32_t r, bool root) {
    if (!isfinite(x)) return 0x7fu;
    uint32_t t = __float_as_uint(fabsf(x) * power(127 - e) * power(kCodeScale)) + r;
    if (root && x > 0.f) t = max(t, 1u << 20);   // what is above zero keeps a code above zero
    return t >> 20 | (root ? 0u : __float_as_uint(x) >> 24 & 0x80u);
}
__device__ __forceinline__ uint32_t finite_bits(float x) {
    const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}

// Where a lane's element k lies in its block: lane l has 4 l .. 4 l + 3 of both halves.
__device__ __forceinline__ int64_t place(int64_t block, int u) { return block * kBlock + u * 128 + (threadIdx.x & 31) * 4; }

__device__ __forceinline__ uint32_t hash_of(uint32_t key, int64_t i) {
    return key + (uint32_t)(i >> 32) * 0xBB67AE85u + (uint32_t)i * 0x9E3779B1u;
}

// One block of 256 elements, by a warp, every operation by itself and element by element: for
// blocks at the ends of tensors, at odd addresses and at the ends of the range.  All loads are in
// flight before the first is used (257 elements: 8.7 us in place of 12.5).
template <typename P, typename G>
__device__ __noinline__ void adamw8_odd_block(const Entry& e, int64_t block, const Hyper& h, const Step& s, uint32_t key) {
    const int64_t n = e.n;
    P* const pp = (P*)e.p;
    uint8_t *const pm = (uint8_t*)e.m, *const pv = (uint8_t*)e.v;
    P p0[8];
    G g0[8];
    uint8_t m0[8], v0[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const int64_t i = place(block, k / 4) + k % 4;
        p0[k] = P(0.f);
        g0[k] = G(0.f);
        m0[k] = v0[k] = 0;
        if (i < n) {
            p0[k] = pp[i];
            g0[k] = ((const G*)e.g)[i];
            m0[k] = pm[i];
            v0[k] = pv[i];
        }
    }
    const float dm = power((int)e.m_exp[block] - 127), ds = power((int)e.v_exp[block] - 127);
    float p[8], m[8], v[8];
    uint32_t tm = 0, tv = 0;
#pragma unroll
    for (int u = 0; u < 2; u++) {
        uint32_t cm = 0, cs = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            cm |= (uint32_t)m0[4 * u + j] << (8 * j);
            cs |= (uint32_t)v0[4 * u + j] << (8 * j);
        }
        decode4(cm, m + 4 * u);
        decode4(cs, v + 4 * u);
#pragma unroll
        for (int j = 4 * u; j < 4 * u + 4; j++) {
            const float gj = __fmul_rn((float)g0[j], s.scale), sj = v[j] * ds;
            m[j] = __fadd_rn(__fmul_rn(m[j] * dm, h.beta1), __fmul_rn(gj, h.rest1));
            v[j] = __fsqrt_rn(__fadd_rn(__fmul_rn(__fmul_rn(sj, sj), h.beta2), __fmul_rn(__fmul_rn(gj, gj), h.rest2)));
            p[j] = stepped((float)p0[j], m[j], v[j], s);
            tm = max(tm, finite_bits(m[j]));
            tv = max(tv, finite_bits(v[j]));
        }
    }
    const int nm = block_exponent(__reduce_max_sync(0xffffffffu, tm));
    const int ns = block_exponent(__reduce_max_sync(0xffffffffu, tv));
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const int64_t i = place(block, k / 4) + k % 4;
        uint32_t rm, rs;
        random_bits(hash_of(key, i), rm, rs);
        if (i < n) {
            store1(pp + i, p[k]);
            pm[i] = (uint8_t)any_code(m[k], nm, rm >> 4, false);
            pv[i] = (uint8_t)any_code(v[k], ns, rs >> 4, true);
            if (e.copy) store1((bf16*)e.copy + i, p[k]);
        }
    }
    if ((threadIdx.x & 31) == 0) {
        e.m_exp[block] = (uint8_t)nm;
        e.v_exp[block] = (uint8_t)ns;
    }
}

// What a step reads of a unit, on its way through shared memory.
template <typename P, typename G>
struct alignas(16) UnitIn {
    P p[kUnit8];
    G g[kUnit8];
    uint8_t m[kUnit8], v[kUnit8];
};

__device__ __forceinline__ void copy16(void* smem, const void* global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
}

// The whole warp copies a unit in, 16 bytes a lane at a time.
template <typename P, typename G>
__device__ __forceinline__ void fetch(UnitIn<P, G>& in, const Entry& e, int unit) {
    const int lane = threadIdx.x & 31;
    auto part = [&](void* to, const void* from, int bytes) {
        const char* at = (const char*)from + (int64_t)unit * bytes + lane * 16;
#pragma unroll
        for (int o = 0; o < bytes; o += 512) copy16((char*)to + o + lane * 16, at + o);
    };
    part(in.p, e.p, sizeof(in.p));
    part(in.g, e.g, sizeof(in.g));
    part(in.m, e.m, sizeof(in.m));
    part(in.v, e.v, sizeof(in.v));
}

// The two blocks of a whole unit at aligned addresses; false, with nothing written, where one is
// not a common one.  The common case folds the exponents into the betas (exact, as they are powers
// of two) and takes the hardware's square root (2^-23), which flushes what is under 2^-126: no code
// depends on its last places there, and the step does only where eps is as small as such a root
// (Step::flushed).
// exps: m's exponents in bytes 0 and 1, s's in 2 and 3.
template <typename P, typename G>
__device__ __forceinline__ bool adamw8_unit(const UnitIn<P, G>& in, uint32_t exps, const Entry& e, int unit, const Hyper& h,
                                            const Step& s, uint32_t key) {
    constexpr int B = 2;
    const int at = (threadIdx.x & 31) * 4;
    const F2 scale2 = f2(s.scale, s.scale), r1 = f2(h.rest1, h.rest1), r2 = f2(h.rest2, h.rest2);
    float m[8 * B], v[8 * B];
    uint32_t tm[B], tv[B];
    bool common = true;
#pragma unroll
    for (int b = 0; b < B; b++) {
        // m beta1 = code * bm and s^2 beta2 = code^2 * bs
        const uint32_t em = exps >> 8 * b & 0xff, es = exps >> 8 * (b + 2) & 0xff;
        const float ds = __uint_as_float(es << 23), bm = __uint_as_float(em << 23) * h.beta1, bs = ds * ds * h.beta2;
        const F2 bm2 = f2(bm, bm), bs2 = f2(bs, bs);
        float top_m = 0.f, top_v = 0.f;
        uint32_t codes = 0;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int o = b * kBlock + u * 128 + at;
            float g[4];
            const uint32_t cm = *(const uint32_t*)(in.m + o), cs = *(const uint32_t*)(in.v + o);
            decode4(cm, m + 8 * b + 4 * u);
            decode4(cs, v + 8 * b + 4 * u);
            codes |= cm | cs;
            load4(in.g + o, g);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const int k = 8 * b + 4 * u + j;
                const F2 g2 = mul(f2(g[j], g[j + 1]), scale2), c2 = f2(v[k], v[k + 1]);
                sums(mul(f2(m[k], m[k + 1]), bm2), mul(g2, r1), m + k);
                sums(mul(mul(c2, c2), bs2), mul(mul(g2, g2), r2), v + k);
                top_m = largest(top_m, m[k], m[k + 1]);
                top_v = largest(top_v, v[k], v[k + 1]);
            }
        }
        tm[b] = __reduce_max_sync(0xffffffffu, __float_as_uint(top_m));
        tv[b] = __reduce_max_sync(0xffffffffu, __float_as_uint(top_v));
        // Moments under 2^14, so that the scale below is a normal number (what is not finite is above); a largest
        // root above 2^-42, next to which a flushed one rounds as its own value does, or none; and held exponents
        // whose products with a code are normal numbers, or codes that are all 0 (a new tensor's).
        common = common && tm[b] < 141u << 23 && tv[b] < 155u << 23 && (tv[b] >= 43u << 23 || tv[b] == 0) &&
                 ((em >= 32 && es >= 84) || __all_sync(0xffffffffu, !codes));
    }
    if (!common) return false;
    if (s.eps <= s.flushed) {
        bool any = s.eps <= 1e-30f;   // what the reciprocal flushes
#pragma unroll
        for (int k = 0; k < 8 * B; k++) any |= v[k] > 0.f && v[k] < 0x1p-126f;
        if (__any_sync(0xffffffffu, any)) return false;
    }
    const F2 root2 = f2(s.root, s.root), eps2 = f2(s.eps, s.eps), rate2 = f2(-s.rate, -s.rate), keep2 = f2(s.keep, s.keep);
    const int64_t i0 = (int64_t)unit * kUnit8 + at;
    const uint32_t hash = hash_of(key, i0);
#pragma unroll
    for (int b = 0; b < B; b++) {
        // exponents of the largest value's binade, less 7; that of a root is half its square's (none rounds up to a
        // power of two)
        const uint32_t nm = max(tm[b] >> 23, 7u) - 7u, ns = tv[b] ? ((tv[b] >> 23) + 113u) >> 1 : 0u;
        const float im = __uint_as_float((134u - nm) << 23), is = __uint_as_float((134u - ns) << 23);   // 2^(127 + kCodeScale - n)
        const F2 im2 = f2(im, im), is2 = f2(is, is);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int o = b * kBlock + u * 128;
            float p[4];
            uint32_t wm[4], ws[4], border = ~0u;
            load4(in.p + o + at, p);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const int k = 8 * b + 4 * u + j;
                const F2 m2 = f2(m[k], m[k + 1]), q2 = f2(sqrt_fast(v[k]), sqrt_fast(v[k + 1]));
                float d[2], x[2], y[2];
                get(fma(q2, root2, eps2), d);
                get(fma(f2(p[j], p[j + 1]), keep2, mul(mul(m2, rate2), f2(rcp_fast(d[0]), rcp_fast(d[1])))), p + j);
                get(mul(m2, im2), x);
                get(mul(q2, is2), y);
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    uint32_t rm, rs;
                    random_bits(hash + (uint32_t)(o + j + w) * 0x9E3779B1u, rm, rs);
                    // 16 x + r: the code's bits 20 to 26 come to 24 to 30, and the sign goes back to 31
                    wm[j + w] = (__float_as_uint(x[w]) * 16u + rm) | (__float_as_uint(x[w]) & 0x80000000u);
                    ws[j + w] = __float_as_uint(y[w]) * 16u + rs;
                    border = min(border, ws[j + w] * 256u + 64u * 256u);
                }
            }
            // Where the root's last two places decide on a code (one element in 100000), the exact one does.
            if (border < 128u * 256u)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    uint32_t rm, rs;
                    random_bits(hash + (uint32_t)(o + j) * 0x9E3779B1u, rm, rs);
                    ws[j] = __float_as_uint(__fsqrt_rn(v[8 * b + 4 * u + j]) * is) * 16u + rs;
                }
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (v[8 * b + 4 * u + j] > 0.f) ws[j] = max(ws[j], 1u << 24);   // what is above zero keeps a code above zero
            store4((P*)e.p + i0 + o, p);
            *(uint32_t*)((uint8_t*)e.m + i0 + o) = top_bytes(wm);
            *(uint32_t*)((uint8_t*)e.v + i0 + o) = top_bytes(ws);
            if (e.copy) store4((bf16*)e.copy + i0 + o, p);
        }
        if ((threadIdx.x & 31) == 0) {
            e.m_exp[(int64_t)unit * 2 + b] = (uint8_t)nm;
            e.v_exp[(int64_t)unit * 2 + b] = (uint8_t)ns;
        }
    }
    return true;
}

// How many units a warp's ring holds and how many CTAs an SM.  With f32 parameters 12 warps
// of 3 or 4 units (5 KB or 4 KB) keep enough in flight for HBM, and more of them cost DRAM
// rows.  With bf16 parameters instruction issue is the bound: as many warps as the registers
// allow.  1e9 parameters, a step by itself / back to back, ms: f32, bf16 gradients and a copy,
// 6 CTAs of 4 units 2.54 / 2.81, 8 of 3 2.91 / 2.72, 10 of 2 2.96 / 2.99, 4 of 4 3.16 / 3.19;
// all bf16, 10 CTAs of 2 units 2.18 / 2.24, 8 of 2 2.20 / 2.25, 10 of 3 2.24 / 2.30, 6 of 4
// 2.39 / 2.35.  An odd number of CTAs leaves sub-partitions of the SM uneven.
template <typename P, typename G>
struct Ring8 {
    static constexpr bool wide = sizeof(P) == 4;
    static constexpr int stages = !wide ? 2 : sizeof(G) == 4 ? 3 : 4;
    static constexpr int ctas = wide ? 6 : 10;
    static_assert(ctas * (sizeof(UnitIn<P, G>) * stages * (kThreads8 / 32) + 1024) <= 227 * 1024, "fits the SM");
};

// Each warp has a ring of units of its own in shared memory: asynchronous copies fill
// the others while it computes one.
template <typename P, typename G, int CAP>
__global__ void __launch_bounds__(kThreads8, Ring8<P, G>::ctas) adamw8_kernel(const __grid_constant__ Table<CAP> t) {
    constexpr int S = Ring8<P, G>::stages;
    __shared__ UnitIn<P, G> rings[kThreads8 / 32][S];
    const int warp = threadIdx.x / 32, chunks = t.start[t.n];
    UnitIn<P, G>* ring = rings[warp];
    auto unit_of = [&](int c, int k) { return (c - t.start[k]) * (kChunk8 / kUnit8) + warp; };
    auto exps_of = [&](int k, int unit) {   // m's in the low half, the first block's in its low byte
        const uint8_t *m = t.e[k].m_exp + (int64_t)unit * 2, *v = t.e[k].v_exp + (int64_t)unit * 2;
        return m[0] | m[1] << 8 | (uint32_t)v[0] << 16 | (uint32_t)v[1] << 24;
    };
    // the units in flight, the present one first
    int ks[S] = {}, units[S] = {};
    uint32_t exps[S] = {};
    bool whole[S] = {};
    int c = blockIdx.x, ahead = c;
    auto start = [&](int i, int stage) {   // the next unit's copies, its place in slot i
        whole[i] = false;
        if (ahead < chunks) {
            ks[i] = i ? advance(t, ks[i - 1], ahead) : find(t, ahead);
            units[i] = unit_of(ahead, ks[i]);
            whole[i] = units[i] < t.whole[ks[i]];
            if (whole[i]) {
                fetch(ring[stage], t.e[ks[i]], units[i]);
                exps[i] = exps_of(ks[i], units[i]);
            }
            ahead += gridDim.x;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < S - 1; i++) start(i, i);
    const Step s = step_of(t.h);
    int known = -1, stage = 0;
    uint32_t key = 0;
    for (; c < chunks; c += gridDim.x) {
        start(S - 1, stage ? stage - 1 : S - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
        __syncwarp();
        const int k = ks[0];
        const Entry& e = t.e[k];
        if (k != known) {
            known = k;
            key = mix(s.key ^ (t.h.first + k));
        }
        if (!(whole[0] && adamw8_unit(ring[stage], exps[0], e, units[0], t.h, s, key))) {
#pragma unroll 1
            for (int64_t block = (int64_t)units[0] * 2; block < (int64_t)units[0] * 2 + 2 && block * kBlock < e.n; block++)
                adamw8_odd_block<P, G>(e, block, t.h, s, key);
        }
        __syncwarp();   // all have read the stage that the next copy fills
        stage = stage + 1 < S ? stage + 1 : 0;
#pragma unroll
        for (int i = 0; i + 1 < S; i++) {
            ks[i] = ks[i + 1];
            units[i] = units[i + 1];
            exps[i] = exps[i + 1];
            whole[i] = whole[i + 1];
        }
    }
}

// -------------------------------------------------------------- grad norm --
// The sum of the squares of 16 bytes, each element times f.
__device__ __forceinline__ float sumsq16(const uint4 a, const float*, float f = 1.f) {
    const float x = __uint_as_float(a.x) * f, y = __uint_as_float(a.y) * f, z = __uint_as_float(a.z) * f,
                w = __uint_as_float(a.w) * f;
    return (x * x + y * y) + (z * z + w * w);
}
__device__ __forceinline__ float sumsq2(uint32_t a, float f) {
    const float x = bf16_lo(a) * f, y = bf16_hi(a) * f;
    return x * x + y * y;
}
__device__ __forceinline__ float sumsq16(const uint4 a, const bf16*, float f = 1.f) {
    return (sumsq2(a.x, f) + sumsq2(a.y, f)) + (sumsq2(a.z, f) + sumsq2(a.w, f));
}

// Whether a thread's sum of squares leaves f32's range at either end: one under 2^-80 may have lost squares to it
// (above that, those under 2^-126 are nothing), one that is not finite may be of finite elements.
__device__ __forceinline__ bool out_of_range(float s) { return !(s > 0x1p-80f && s < INFINITY); }
// What takes the elements of such a sum to where f32 holds their squares, exactly, as it is a power of two; the sum's
// own factor is its square's inverse.
__device__ __forceinline__ float range_factor(float s) { return s < 1.f ? 0x1p100f : 0x1p-100f; }
__device__ __forceinline__ double from_range(float s, float f) { return (double)s * (f > 1.f ? 0x1p-200 : 0x1p200); }

// part[blockIdx.x] = the CTA's sum of squares: f32 over a chunk's 32 elements a
// thread, f64 over the chunks.  All of a chunk's loads are in flight at once.
// Where f32 does not hold the squares, the elements are taken again, scaled.
template <typename G, int CAP>
__global__ void __launch_bounds__(kThreads) sumsq_kernel(const __grid_constant__ Table<CAP> t, double* __restrict__ part) {
    constexpr int V = 16 / sizeof(G), L = kNormChunk / kThreads / V;
    __shared__ double red[kThreads / 32];
    const int chunks = t.start[t.n];
    double acc = 0.0;
    int k = find(t, blockIdx.x);
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        k = advance(t, k, c);
        const G* g = (const G*)t.e[k].g;
        const int64_t i0 = (int64_t)(c - t.start[k]) * kNormChunk, n = t.e[k].n;
        float s = 0.f;
        if (t.vec[k] && i0 + kNormChunk <= n) {
            uint4 a[L];
#pragma unroll
            for (int u = 0; u < L; u++) a[u] = *reinterpret_cast<const uint4*>(g + i0 + (u * kThreads + threadIdx.x) * V);
#pragma unroll
            for (int u = 0; u < L; u++) s += sumsq16(a[u], g);
            if (out_of_range(s)) {
                const float f = range_factor(s);
                s = 0.f;
#pragma unroll
                for (int u = 0; u < L; u++) s += sumsq16(a[u], g, f);
                acc += from_range(s, f);
                continue;
            }
        } else {
#pragma unroll 8
            for (int64_t i = i0 + threadIdx.x; i < n && i < i0 + kNormChunk; i += kThreads) {
                const float x = load1(g + i);
                s += x * x;
            }
            if (out_of_range(s)) {
                const float f = range_factor(s);
                s = 0.f;
                for (int64_t i = i0 + threadIdx.x; i < n && i < i0 + kNormChunk; i += kThreads) {
                    const float x = load1(g + i) * f;
                    s += x * x;
                }
                acc += from_range(s, f);
                continue;
            }
        }
        acc += s;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kThreads / 32; w++) acc += red[w];
        part[blockIdx.x] = acc;
    }
}

// norm = sqrt(sum of the parts), in a fixed order; scale = min(1, max_norm / (norm + 1e-6)).
__global__ void __launch_bounds__(kThreads) norm_kernel(const double* __restrict__ part, int n, float* __restrict__ norm,
                                                        float* __restrict__ scale, double max_norm) {
    __shared__ double red[kThreads / 32];
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) acc += part[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = acc;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < kThreads / 32; w++) acc += red[w];
    acc = sqrt(acc);
    *norm = (float)acc;
    // a norm that is not a number gives a scale that is none
    const double f = max_norm / (acc + 1e-6);
    if (scale) *scale = f > 1.0 ? 1.f : (float)f;
}

// ------------------------------------------------------------------- host --
int64_t chunks_of(int64_t n, int chunk) { return (n + chunk - 1) / chunk; }

// Elements in a list at most, so that chunks and units are counted in 32 bits.
constexpr int64_t kMostElements = 1ll << 39;

// Fills a table with the first tensors of a list; returns its chunks.
template <int CAP>
int fill(Table<CAP>& t, const Entry* e, const uint8_t* vec, int count, int chunk) {
    t.n = count;
    t.start[0] = 0;
    for (int k = 0; k < count; k++) {
        t.e[k] = e[k];
        t.vec[k] = vec[k];
        t.whole[k] = vec[k] ? (int)(e[k].n / kUnit8) : 0;
        t.start[k + 1] = t.start[k] + (int)chunks_of(e[k].n, chunk);
    }
    return t.start[count];
}

unsigned grid_for(tb_ctx* ctx, int64_t chunks, int ctas = kCtasPerSm) {
    const int64_t cap = (int64_t)ctx->num_sms * ctas;
    return (unsigned)(chunks < cap ? chunks : cap);
}

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

template <typename P, typename G, int CAP>
int adamw_launch(tb_ctx* ctx, int bits, const Entry* e, const uint8_t* vec, int count, const Hyper& h) {
    Table<CAP> t;
    const int chunks = fill(t, e, vec, count, bits == 8 ? kChunk8 : kChunk);
    if (!chunks) return TB_OK;
    t.h = h;
    if (bits == 8)
        return launch(ctx, "adamw8", adamw8_kernel<P, G, CAP>, dim3(grid_for(ctx, chunks, Ring8<P, G>::ctas)), dim3(kThreads8), 0,
                      t);
    return launch(ctx, "adamw", adamw_kernel<P, G, CAP>, dim3(grid_for(ctx, chunks, adamw_ctas<P, G>())), dim3(kThreads), 0, t);
}

template <typename G, int CAP>
int sumsq_launch(tb_ctx* ctx, const Entry* e, const uint8_t* vec, int count, double* part) {
    Table<CAP> t;
    const int chunks = fill(t, e, vec, count, kNormChunk);
    t.h = Hyper{};
    // every launch writes its own row of partial sums, of one CTA where there is nothing to add
    return launch(ctx, "grad_norm", sumsq_kernel<G, CAP>, dim3(chunks ? grid_for(ctx, chunks) : 1u), dim3(kThreads), 0, t,
                  part);
}

int launches_of(int n) { return n <= kSmallTable ? 1 : (n + kLargeTable - 1) / kLargeTable; }

}  // namespace
}  // namespace tb

using namespace tb;

struct tb_adamw {
    tb_ctx* ctx = nullptr;
    int p_dtype = 0, g_dtype = 0, bits = 32, n = 0;
    Entry* e = nullptr;
    uint8_t* vec = nullptr;
};

namespace tb {
namespace {

struct Range {
    uintptr_t lo, hi;
    bool written;
};

// Whether two ranges meet of which one is written.
bool overlap(Range* r, size_t n) {
    std::sort(r, r + n, [](const Range& a, const Range& b) { return a.lo < b.lo; });
    uintptr_t written = 0, any = 0;
    for (size_t i = 0; i < n; i++) {
        if (r[i].lo < (r[i].written ? any : written)) return true;
        any = std::max(any, r[i].hi);
        if (r[i].written) written = std::max(written, r[i].hi);
    }
    return false;
}

}  // namespace
}  // namespace tb

extern "C" {

int tb_adamw_create(tb_ctx* ctx, int p_dtype, int g_dtype, int state_bits, const tb_adamw_tensor* tensors, int n,
                    tb_adamw** out) {
    if (!out) return TB_ERR_ARG;
    *out = nullptr;
    if (!ctx) return TB_ERR_ARG;
    TB_REQUIRE(ctx, n >= 0 && (n == 0 || tensors), TB_ERR_ARG, "adamw: bad list of tensors");
    const bool types = (p_dtype == TB_F32 && (g_dtype == TB_F32 || g_dtype == TB_BF16)) ||
                       (p_dtype == TB_BF16 && g_dtype == TB_BF16);
    TB_REQUIRE(ctx, types, TB_ERR_UNSUPPORTED, "adamw: parameters and gradients f32 / f32, f32 / bf16 or bf16 / bf16");
    TB_REQUIRE(ctx, state_bits == 32 || state_bits == 8, TB_ERR_UNSUPPORTED, "adamw: moments in 32 or 8 bits");
    const size_t ps = p_dtype == TB_F32 ? 4 : 2, gs = g_dtype == TB_F32 ? 4 : 2, ms = state_bits / 8;
    int64_t total = 0;
    for (int k = 0; k < n; k++) {
        const tb_adamw_tensor& t = tensors[k];
        TB_REQUIRE(ctx, t.n >= 0 && t.n <= kMostElements - total, TB_ERR_SHAPE, "adamw: tensor %d has %lld elements", k,
                   (long long)t.n);
        total += t.n;
        if (!t.n) continue;
        TB_REQUIRE(ctx, t.p && t.g && t.m && t.v && (state_bits == 32 || (t.m_exp && t.v_exp)), TB_ERR_ARG,
                   "adamw: null pointer in tensor %d", k);
        TB_REQUIRE(ctx, aligned(t.p, ps) && aligned(t.g, gs) && aligned(t.m, ms) && aligned(t.v, ms) &&
                            aligned(t.copy, 2),
                   TB_ERR_ALIGN, "adamw: tensor %d is not aligned to its type", k);
        TB_REQUIRE(ctx, !t.copy || p_dtype == TB_F32, TB_ERR_UNSUPPORTED, "adamw: a bf16 copy goes with f32 parameters");
    }
    tb_adamw* a = new (std::nothrow) tb_adamw();
    Range* r = (Range*)malloc(sizeof(Range) * 7 * (size_t)(n + 1));
    if (a) {
        a->e = (Entry*)malloc(sizeof(Entry) * (size_t)(n + 1));
        a->vec = (uint8_t*)malloc((size_t)(n + 1));
    }
    if (!a || !r || !a->e || !a->vec) {
        free(r);
        tb_adamw_destroy(a);
        return set_error(ctx, TB_ERR_OOM, "adamw: out of host memory");
    }
    a->ctx = ctx;
    a->p_dtype = p_dtype;
    a->g_dtype = g_dtype;
    a->bits = state_bits;
    a->n = n;
    size_t nr = 0;
    auto add = [&](const void* p, size_t bytes, bool written) {
        if (p && bytes) r[nr++] = {(uintptr_t)p, (uintptr_t)p + bytes, written};
    };
    for (int k = 0; k < n; k++) {
        const tb_adamw_tensor& t = tensors[k];
        a->e[k] = {t.p, t.g, t.m, t.v, t.m_exp, t.v_exp, t.copy, t.n};
        // four elements at a time; 16 bytes where blocks go through shared memory
        a->vec[k] = state_bits == 8 ? aligned16(t.p) && aligned16(t.g) && aligned16(t.m) && aligned16(t.v) && aligned(t.copy, 8)
                                    : aligned(t.p, 4 * ps) && aligned(t.g, 4 * gs) && aligned16(t.m) && aligned16(t.v) &&
                                          aligned(t.copy, 8);
        const size_t cnt = (size_t)t.n, blocks = (cnt + kBlock - 1) / kBlock;
        add(t.p, cnt * ps, true);
        add(t.g, cnt * gs, false);
        add(t.m, cnt * ms, true);
        add(t.v, cnt * ms, true);
        add(t.copy, cnt * 2, true);
        if (state_bits == 8) {
            add(t.m_exp, blocks, true);
            add(t.v_exp, blocks, true);
        }
    }
    const bool bad = overlap(r, nr);
    free(r);
    if (bad) {
        tb_adamw_destroy(a);
        return set_error(ctx, TB_ERR_ARG, "adamw: tensors overlap (a parameter listed twice, or memory shared)");
    }
    *out = a;
    return TB_OK;
}

int tb_adamw_destroy(tb_adamw* a) {
    if (!a) return TB_OK;
    free(a->e);
    free(a->vec);
    delete a;
    return TB_OK;
}

int tb_adamw_step(tb_adamw* a, const tb_adamw_hyper* hy) {
    if (!a) return TB_ERR_ARG;
    tb_ctx* ctx = a->ctx;
    TB_REQUIRE(ctx, hy, TB_ERR_ARG, "adamw: null pointer");
    // written so that a NaN fails each of them
    TB_REQUIRE(ctx, hy->beta1 >= 0 && hy->beta1 < 1 && hy->beta2 >= 0 && hy->beta2 < 1 && hy->eps >= 0 &&
                        hy->weight_decay >= 0 && (hy->lr_dev || hy->lr >= 0),
               TB_ERR_ARG, "adamw: betas in [0, 1), lr, eps and weight_decay >= 0");
    TB_REQUIRE(ctx, hy->step_dev || hy->step >= 1, TB_ERR_ARG, "adamw: steps count from 1");
    TB_REQUIRE(ctx, aligned(hy->lr_dev, 4) && aligned(hy->grad_scale, 4) && aligned(hy->step_dev, 8), TB_ERR_ALIGN,
               "adamw: a scalar is not aligned to its type");
    Hyper h = {};
    h.lr = (float)hy->lr;
    h.beta1 = (float)hy->beta1;
    h.beta2 = (float)hy->beta2;
    h.rest1 = (float)(1.0 - hy->beta1);
    h.rest2 = (float)(1.0 - hy->beta2);
    // The division flushes a divisor under 2^-126, so an eps above 0 is at least that: 0 / eps stays 0, and next to a
    // root above 0 (2^-75 at least, that of f32's smallest number) neither is seen.
    h.eps = hy->eps > 0 ? std::max((float)hy->eps, FLT_MIN) : 0.f;
    h.decay = (float)hy->weight_decay;
    h.log1 = (float)log(hy->beta1);   // -inf for 0: the correction is 1
    h.log2 = (float)log(hy->beta2);
    h.step = hy->step;
    h.lr_dev = hy->lr_dev;
    h.grad_scale = hy->grad_scale;
    h.step_dev = hy->step_dev;
    h.seed = (uint32_t)hy->seed;
    const int cap = a->n <= kSmallTable ? kSmallTable : kLargeTable;
    for (int at = 0; at < a->n; at += cap) {
        const int count = std::min(cap, a->n - at);
        h.first = (uint32_t)at;
        auto go = [&](auto small, auto large) {
            return cap == kSmallTable ? small(ctx, a->bits, a->e + at, a->vec + at, count, h)
                                      : large(ctx, a->bits, a->e + at, a->vec + at, count, h);
        };
        const int rc = a->p_dtype == TB_BF16   ? go(adamw_launch<bf16, bf16, kSmallTable>, adamw_launch<bf16, bf16, kLargeTable>)
                       : a->g_dtype == TB_BF16 ? go(adamw_launch<float, bf16, kSmallTable>, adamw_launch<float, bf16, kLargeTable>)
                                               : go(adamw_launch<float, float, kSmallTable>, adamw_launch<float, float, kLargeTable>);
        if (rc) return rc;
    }
    return TB_OK;
}

size_t tb_grad_norm_ws(int64_t n) {
    // a row of partial sums for each launch: CTAs for 160 SMs
    return n < 0 || n >= (1ll << 31) ? 0 : (size_t)launches_of((int)n) * 160 * kCtasPerSm * 8;
}

int tb_grad_norm(tb_ctx* ctx, int dtype, const void* const* grads, const int64_t* sizes, int n, float* norm, float* scale,
                 double max_norm, void* workspace, size_t workspace_bytes) {
    if (!ctx) return TB_ERR_ARG;
    TB_REQUIRE(ctx, n >= 0 && (n == 0 || (grads && sizes)) && norm, TB_ERR_ARG, "grad_norm: null pointer");
    if (dtype != TB_F32 && dtype != TB_BF16) return set_error(ctx, TB_ERR_UNSUPPORTED, "grad_norm: dtype %d", dtype);
    TB_REQUIRE(ctx, !scale || max_norm >= 0, TB_ERR_ARG, "grad_norm: max_norm >= 0");
    const size_t es = dtype == TB_F32 ? 4 : 2;
    int64_t total = 0;
    for (int k = 0; k < n; k++) {
        TB_REQUIRE(ctx, sizes[k] >= 0 && sizes[k] <= kMostElements - total, TB_ERR_SHAPE, "grad_norm: tensor %d has %lld elements",
                   k, (long long)sizes[k]);
        total += sizes[k];
        TB_REQUIRE(ctx, grads[k] || !sizes[k], TB_ERR_ARG, "grad_norm: null pointer");
        TB_REQUIRE(ctx, aligned(grads[k], es), TB_ERR_ALIGN, "grad_norm: tensor %d is not aligned to its type", k);
    }
    const size_t need = tb_grad_norm_ws(n);
    TB_REQUIRE(ctx, workspace && workspace_bytes >= need && aligned(workspace, 8), TB_ERR_ARG,
               "grad_norm: workspace of %zu bytes required (tb_workspace_bytes)", need);
    TB_REQUIRE(ctx, ctx->num_sms <= 160, TB_ERR_UNSUPPORTED, "grad_norm: more SMs than the workspace is made for");
    double* part = (double*)workspace;
    const int cap = n <= kSmallTable ? kSmallTable : kLargeTable;
    int parts = 0;
    for (int at = 0; at < n || at == 0; at += cap) {
        const int count = std::min(cap, n - at);
        Entry e[kLargeTable];
        uint8_t vec[kLargeTable];
        int64_t chunks = 0;
        for (int k = 0; k < count; k++) {
            e[k] = Entry{};
            e[k].g = grads[at + k];
            e[k].n = sizes[at + k];
            vec[k] = aligned16(e[k].g);
            chunks += chunks_of(e[k].n, kNormChunk);
        }
        auto go = [&](auto small, auto large) {
            return cap == kSmallTable ? small(ctx, e, vec, count, part + parts) : large(ctx, e, vec, count, part + parts);
        };
        const int rc = dtype == TB_F32 ? go(sumsq_launch<float, kSmallTable>, sumsq_launch<float, kLargeTable>)
                                       : go(sumsq_launch<bf16, kSmallTable>, sumsq_launch<bf16, kLargeTable>);
        if (rc) return rc;
        parts += chunks ? (int)grid_for(ctx, chunks) : 1;
    }
    return launch(ctx, "grad_norm_final", norm_kernel, dim3(1), dim3(kThreads), 0, (const double*)part, parts, norm, scale,
                  max_norm);
}

}  // extern "C"
