// LayerNorm for training: the forward that keeps each row's mean and rstd, and
// the backward with the reduction of the weight's and the bias's gradients
// (the reference's layer_norm_forward, nn/norm/layernorm.rs:163).
//
//   y = xhat w + b,  xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)
//   a = dy w,  c1 = sum_n(a) / N,  c2 = sum_n(a xhat) / N
//   dx = rstd (a - c1 - xhat c2),  dw = sum_m dy xhat,  db = sum_m dy
//
// Bound by HBM: the forward moves x and y, the backward x, dy and dx, once
// each.  A row belongs to a group of threads (a warp, or a CTA of as many as the
// row needs), 16 elements a thread (two 16-byte vectors of bf16, four of f32); the
// groups walk the rows with the grid's stride and keep w (and b) in registers.
// Each thread copies its own vectors of the next rows into its own slots of a ring
// in shared memory (cp.async: no registers, no barrier), so that rows are in flight
// while one is reduced.  In the backward each thread also keeps the f32 sums of dw
// and db for its columns over all the rows it walks; the CTAs write them as partial
// rows, and a second launch adds those in CTA order: no atomics, the same bits on
// each run.
//
// Rows whose length is no multiple of a vector start at any element.  Their
// vectors are those of the tensor: the first may begin in the row before, the last
// ends where the row does.  What a row's start is off a vector's is the same for
// all rows of a group, since the grid's stride is a multiple of its period.
//
// Rows longer than a CTA's registers hold (8192 elements), and tensors that do not
// start at 16 bytes, take the `wide` kernels: a CTA a row, which registers hold up
// to 16384 elements, else passes over it; dw and db in a launch of their own.
//
// Measured on the device (inputs larger than L2; the floor is the bytes at the rate
// of a copy, 6.45 TB/s): forward 16384 x 2048 bf16 21.6 us (floor 20.8), 4096 x 8192
// f32 47 (41.6), 3001 x 5003 bf16 18 (9.3), 128 x 256 f32 2.1; backward 16384 x 2048
// bf16 41.2 (31.2), of which 8 are the start and the sums of partial rows, 65536 x
// 2048 145 (124.8), 2047 x 8192 f32 37.5 (31.2), 3001 x 5003 bf16 38 (14.0), 128 x
// 256 f32 5.6.  What bounds the backward is the latency of a row's sums (shuffles,
// barrier, shared memory) at the 16 warps that 128 registers a thread leave an SM:
// two rows a barrier, or the next row's first half beside this one's second, cost
// more instructions than they hid (47 us), and so did 24 warps that read a row twice
// from the ring (54 us).
#include <math.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "f32x2.cuh"
#include "rowvec.cuh"

namespace tb {
namespace {

using bf16 = __nv_bfloat16;

constexpr int64_t kLnMaxCols = 8192;   // longer rows: the kernels of several passes
constexpr int kLnStages = 3;           // rows in a ring, one of them being computed
constexpr int kLnSms = 148;            // grids are functions of the shape alone, as the workspace is

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Barrier of a group of NT consecutive threads, of R in the CTA.  A barrier whose number
// is not a constant takes all 16 of a CTA, and four such CTAs all of an SM.
template <int NT, int R>
__device__ __forceinline__ void group_sync() {
    if (R == 1) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + threadIdx.x / NT), "n"(NT) : "memory");
}
// Sums over a group; red has an entry for each of the CTA's warps.  The caller alternates
// two of them: a thread that writes one again has passed the barrier of the other, which
// every reader of the first has reached.
template <int NT, int R>
__device__ __forceinline__ float group_sum(float v, float2* red) {
    v = warp_sum(v);
    if (NT == 32) return v;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32].x = v;
    group_sync<NT, R>();
    if (R > 1) red += threadIdx.x / NT * (NT / 32);
    v = red[0].x;
#pragma unroll
    for (int w = 1; w < NT / 32; w++) v += red[w].x;
    return v;
}
// Both sums in the shuffles of one and a half: the halves of the warp take one each.
template <int NT, int R>
__device__ __forceinline__ float2 group_sum2(float a, float b, float2* red) {
    const bool high = threadIdx.x & 16;
    float v = (high ? b : a) + __shfl_xor_sync(0xffffffffu, high ? a : b, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const float other = __shfl_xor_sync(0xffffffffu, v, 16);
    float2 s = high ? make_float2(other, v) : make_float2(v, other);
    if (NT == 32) return s;
    if ((threadIdx.x & 31) == 0) red[threadIdx.x / 32] = s;
    group_sync<NT, R>();
    if (R > 1) red += threadIdx.x / NT * (NT / 32);
    s = red[0];
#pragma unroll
    for (int w = 1; w < NT / 32; w++) {
        const float2 r = red[w];
        s.x += r.x;
        s.y += r.y;
    }
    return s;
}

// src_bytes of 16 from global memory, zeros behind them.
__device__ __forceinline__ void copy16(uint4* smem, const void* global, int src_bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(smem)), "l"(global), "r"(src_bytes) : "memory");
}
__device__ __forceinline__ void copy4(float* smem, const float* global) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A thread's columns of the rows of its group: VPT vectors of V, NT vectors apart.
// SHIFT: rows may start inside a vector.
template <typename T, int VPT, int NT, bool SHIFT>
struct Cols {
    static constexpr int V = 16 / sizeof(T), P = V / 2;
    int c0, N;   // first column of the first vector; under 0 where it begins in the row before
    // off: elements from a vector's start to the row's
    __device__ __forceinline__ Cols(int N_, int off, int t) : c0(t * V - off), N(N_) {}
    __device__ __forceinline__ int col(int i) const { return c0 + i * NT * V; }
    __device__ __forceinline__ bool any(int i) const { return col(i) < N; }
    __device__ __forceinline__ bool part(int i) const { return SHIFT && (col(i) < 0 || col(i) + V > N); }
    __device__ __forceinline__ bool has(int i, int j) const { return (!SHIFT || col(i) + j >= 0) && col(i) + j < N; }
    // a row's vector i into a slot; row points at column c0
    __device__ __forceinline__ void copy(uint4* slot, const T* row, int i) const {
        if (any(i)) copy16(slot, row + i * NT * V, SHIFT && col(i) + V > N ? (N - col(i)) * (int)sizeof(T) : 16);
    }
    // what is not the row's as 0; a branch of its own, as few warps have such a vector
    __device__ __forceinline__ void mask(int i, F2* v) const {
        if (part(i)) {
            asm volatile("" ::: "memory");
#pragma unroll
            for (int j = 0; j < P; j++) {
                float e[2];
                get(v[j], e);
                v[j] = f2(has(i, 2 * j) ? e[0] : 0.f, has(i, 2 * j + 1) ? e[1] : 0.f);
            }
        }
    }
    // zeros in the slots of vectors that no row has
    __device__ __forceinline__ void clear(uint4* slot, int i) const {
        if (!any(i)) *slot = make_uint4(0, 0, 0, 0);
    }
    // the slot's values, as pairs
    __device__ __forceinline__ void load(const uint4* slot, int i, F2* v) const {
        RowVec<T, V> r;
        r.load(reinterpret_cast<const T*>(slot));
#pragma unroll
        for (int j = 0; j < P; j++) v[j] = f2(r.get(2 * j), r.get(2 * j + 1));
        mask(i, v);
    }
    __device__ __forceinline__ void store(T* row, int i, const F2* v) const {
        float e[V];
#pragma unroll
        for (int j = 0; j < P; j++) get(v[j], e + 2 * j);
        if (part(i)) {
#pragma unroll
            for (int j = 0; j < V; j++)
                if (has(i, j)) RowVec<T, 1>::store(row + i * NT * V + j, e + j);
        } else if (any(i)) {
            RowVec<T, V>::store(row + i * NT * V, e);
        }
    }
    // a parameter (w, b) once, at any address
    __device__ __forceinline__ void load_param(const T* p, F2* v) const {
        if (!SHIFT && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < VPT; i++) {
                RowVec<T, V> a;
                a.zero();
                if (any(i)) a.load(p + col(i));
#pragma unroll
                for (int j = 0; j < P; j++) v[i * P + j] = f2(a.get(2 * j), a.get(2 * j + 1));
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < VPT; i++)
#pragma unroll
            for (int j = 0; j < P; j++) {
                RowVec<T, 1> a, b;
                a.zero();
                b.zero();
                if (has(i, 2 * j)) a.load(p + col(i) + 2 * j);
                if (has(i, 2 * j + 1)) b.load(p + col(i) + 2 * j + 1);
                v[i * P + j] = f2(a.get(0), b.get(0));
            }
    }
};

// Elements from the last vector's start to row m's.
template <typename T>
__device__ __forceinline__ int row_offset(int64_t m, int N) {
    return (int)((uint64_t)m * (uint64_t)N % (16 / sizeof(T)));
}

// Threads of a CTA: the forward's groups are CTAs of their own (warps go eight to one), the
// backward's share one as large as registers allow, whose groups add their sums of dw and db
// in shared memory first.
template <int NT>
constexpr int fwd_cta() { return NT == 32 ? 256 : NT; }
template <int NT>
constexpr int bwd_cta() { return NT % 3 ? 512 : 384; }

// ---------------------------------------------------------------- forward --
template <typename T, int VPT, int NT, bool SHIFT>
__global__ void __launch_bounds__(fwd_cta<NT>()) ln_fwd_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                              const T* __restrict__ b, T* __restrict__ y,
                                                              float* __restrict__ mean, float* __restrict__ rstd, int64_t M,
                                                              int N, float eps) {
    using C = Cols<T, VPT, NT, SHIFT>;
    constexpr int P = C::P, K = P * VPT, S = kLnStages, CTA = fwd_cta<NT>(), R = CTA / NT;
    extern __shared__ uint4 ring[];   // [S][VPT][CTA]
    __shared__ float2 red[2][CTA / 32];
    const int t = threadIdx.x % NT;
    const int64_t first = (int64_t)blockIdx.x * R + threadIdx.x / NT, stride = (int64_t)gridDim.x * R;
    if (first >= M) return;   // the whole group
    const C cols(N, SHIFT ? row_offset<T>(first, N) : 0, t);
    const int64_t step = stride * N;
    const T* xp = x + first * N + cols.c0;   // of the next row to fetch
    T* yp = y + first * N + cols.c0;
    int ahead = (int)((M - first + stride - 1) / stride);   // rows left to fetch
    auto fetch = [&](uint4* slot) {
        if (ahead-- > 0)
#pragma unroll
            for (int i = 0; i < VPT; i++) cols.copy(slot + i * CTA, xp, i);
        copy_commit();
        xp += step;
    };
    uint4* const base = ring + threadIdx.x;
#pragma unroll
    for (int s = 0; s < S * VPT; s++) cols.clear(base + s * CTA, s % VPT);
#pragma unroll
    for (int s = 0; s < S - 1; s++) fetch(base + s * VPT * CTA);
    F2 wv[K], bv[K];
    cols.load_param(w, wv);
    cols.load_param(b, bv);
    const float inv = 1.f / (float)N;
    uint4 *slot = base, *last = base + (S - 1) * VPT * CTA;
    for (int64_t row = first; row < M; row += stride) {
        fetch(last);
        copy_wait<S - 1>();
        F2 v[K], sum = f2(0.f);
        float e[2];
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            cols.load(slot + i * CTA, i, v + i * P);
#pragma unroll
            for (int j = 0; j < P; j++) sum = add(sum, v[i * P + j]);
        }
        last = slot;
        slot = slot + VPT * CTA < base + S * VPT * CTA ? slot + VPT * CTA : base;
        get(sum, e);
        const float mu = group_sum<NT, R>(e[0] + e[1], red[0]) * inv;
        const F2 minus = f2(-mu);
        F2 q = f2(0.f);
#pragma unroll
        for (int i = 0; i < VPT; i++) {
#pragma unroll
            for (int j = 0; j < P; j++) v[i * P + j] = add(v[i * P + j], minus);
            if (SHIFT) cols.mask(i, v + i * P);
            if (cols.any(i))
#pragma unroll
                for (int j = 0; j < P; j++) q = fma(v[i * P + j], v[i * P + j], q);
        }
        get(q, e);
        const float rs = rsqrtf(group_sum<NT, R>(e[0] + e[1], red[1]) * inv + eps);
        const F2 rs2 = f2(rs);
#pragma unroll
        for (int i = 0; i < VPT; i++) {
#pragma unroll
            for (int j = 0; j < P; j++) v[i * P + j] = fma(mul(v[i * P + j], rs2), wv[i * P + j], bv[i * P + j]);
            cols.store(yp, i, v + i * P);
        }
        yp += step;
        if (t == 0) {
            mean[row] = mu;
            rstd[row] = rs;
        }
    }
}

// Any row: one CTA of 1024.  K > 0: K vectors a thread hold it; else three passes (the second
// and third find the row in L2).
constexpr int kWide = 1024;

// f(vector, its first column) for a thread's vectors of a row.
template <typename T, int V, int K, typename F>
__device__ __forceinline__ void each_vector(int64_t N, F f) {
    if (K) {
#pragma unroll
        for (int i = 0; i < K; i++) {
            const int64_t c = (int64_t)(i * kWide + threadIdx.x) * V;
            if (c < N) f(i, c);
        }
    } else {
        for (int64_t c = (int64_t)threadIdx.x * V; c < N; c += kWide * V) f(0, c);
    }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(kWide) ln_fwd_wide_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                            const T* __restrict__ b, T* __restrict__ y,
                                                            float* __restrict__ mean, float* __restrict__ rstd, int64_t N,
                                                            float eps) {
    __shared__ float2 red[2][32];
    const T* xr = x + (int64_t)blockIdx.x * N;
    T* yr = y + (int64_t)blockIdx.x * N;
    const float inv = 1.f / (float)N;
    RowVec<T, V> v[K ? K : 1];
    float s = 0.f;
    if (K) each_vector<T, V, K>(N, [&](int i, int64_t c) { v[i].load(xr + c); });   // all in flight
    each_vector<T, V, K>(N, [&](int i, int64_t c) {
        if (!K) v[0].load(xr + c);
#pragma unroll
        for (int j = 0; j < V; j++) s += v[i].get(j);
    });
    const float mu = group_sum<kWide, 1>(s, red[0]) * inv;
    float q = 0.f;
    each_vector<T, V, K>(N, [&](int i, int64_t c) {
        if (!K) v[0].load(xr + c);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float d = v[i].get(j) - mu;
            q += d * d;
        }
    });
    const float rs = rsqrtf(group_sum<kWide, 1>(q, red[1]) * inv + eps);
    each_vector<T, V, K>(N, [&](int i, int64_t c) {
        RowVec<T, V> g, h;
        if (!K) v[0].load(xr + c);
        g.load(w + c);
        h.load(b + c);
        float o[V];
#pragma unroll
        for (int j = 0; j < V; j++) o[j] = (v[i].get(j) - mu) * rs * g.get(j) + h.get(j);
        RowVec<T, V>::store(yr + c, o);
    });
    if (threadIdx.x == 0) {
        mean[blockIdx.x] = mu;
        rstd[blockIdx.x] = rs;
    }
}

// --------------------------------------------------------------- backward --
// Where a launch's sums of dw and db go: row k of part, [2][N] each, or, of one CTA alone, the results.
struct Sums {
    float *part, *dw, *db;
    int64_t N;
    int accumulate;
    __device__ __forceinline__ void put(int64_t k, int64_t rows, int64_t c, float v) const {
        if (rows > 1) {
            part[k * 2 * N + c] = v;
            return;
        }
        float* out = c < N ? dw + c : db + (c - N);
        *out = accumulate ? *out + v : v;
    }
};

template <typename T, int VPT, int NT, bool SHIFT>
__global__ void __launch_bounds__(bwd_cta<NT>()) ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                              const T* __restrict__ w, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, T* __restrict__ dx,
                                                              const Sums out, int64_t M, int N) {
    using C = Cols<T, VPT, NT, SHIFT>;
    constexpr int P = C::P, K = P * VPT, S = kLnStages, CTA = bwd_cta<NT>(), R = CTA / NT;
    extern __shared__ uint4 ring[];   // [S][x, dy][VPT][CTA]
    __shared__ float2 stats[S][CTA];  // each thread's copies of mean and rstd
    __shared__ float2 red[2][CTA / 32];
    const int t = threadIdx.x % NT;
    const int64_t first = (int64_t)blockIdx.x * R + threadIdx.x / NT, stride = (int64_t)gridDim.x * R;
    const C cols(N, SHIFT ? row_offset<T>(first, N) : 0, t);
    const int64_t step = stride * N;
    const T *xp = x + first * N + cols.c0, *gp = dy + first * N + cols.c0;   // of the next row to fetch
    T* op = dx + first * N + cols.c0;
    int left = first < M ? (int)((M - first + stride - 1) / stride) : 0, ahead = left;   // rows; rows to fetch
    const float *mp = mean + first, *rp = rstd + first;
    auto fetch = [&](int s) {
        if (ahead-- > 0) {
            uint4* slot = ring + s * 2 * VPT * CTA + threadIdx.x;
#pragma unroll
            for (int i = 0; i < VPT; i++) {
                cols.copy(slot + i * CTA, xp, i);
                cols.copy(slot + (VPT + i) * CTA, gp, i);
            }
            copy4(&stats[s][threadIdx.x].x, mp);
            copy4(&stats[s][threadIdx.x].y, rp);
        }
        copy_commit();
        xp += step;
        gp += step;
        mp += stride;
        rp += stride;
    };
#pragma unroll
    for (int s = 0; s < S * 2 * VPT; s++) cols.clear(ring + s * CTA + threadIdx.x, s % VPT);
#pragma unroll
    for (int s = 0; s < S - 1; s++) fetch(s);
    F2 wv[K], aw[K], ab[K];
    cols.load_param(w, wv);
#pragma unroll
    for (int k = 0; k < K; k++) aw[k] = ab[k] = f2(0.f);
    const float inv = 1.f / (float)N;
    int s = 0, buf = 0;
    for (; left > 0; left--) {
        fetch(s ? s - 1 : S - 1);
        copy_wait<S - 1>();
        const uint4* slot = ring + s * 2 * VPT * CTA + threadIdx.x;
        const float mu = stats[s][threadIdx.x].x, rs = stats[s][threadIdx.x].y;
        F2 xh[K], a[K], sa = f2(0.f), sx = f2(0.f);
        const F2 minus = f2(-mu), r = f2(rs);
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            cols.load(slot + i * CTA, i, xh + i * P);
            cols.load(slot + (VPT + i) * CTA, i, a + i * P);
#pragma unroll
            for (int k = i * P; k < i * P + P; k++) {
                xh[k] = mul(add(xh[k], minus), r);
                aw[k] = fma(a[k], xh[k], aw[k]);
                ab[k] = add(ab[k], a[k]);
                a[k] = mul(a[k], wv[k]);
                sa = add(sa, a[k]);
                sx = fma(a[k], xh[k], sx);
            }
        }
        s = s + 1 < S ? s + 1 : 0;
        float e[2], f[2];
        get(sa, e);
        get(sx, f);
        const float2 sum = group_sum2<NT, R>(e[0] + e[1], f[0] + f[1], red[buf]);
        buf ^= 1;
        const F2 k1 = f2(-sum.x * inv * rs), k2 = f2(-sum.y * inv * rs);
#pragma unroll
        for (int i = 0; i < VPT; i++) {
#pragma unroll
            for (int k = i * P; k < i * P + P; k++) a[k] = fma(xh[k], k2, fma(a[k], r, k1));
            cols.store(op, i, a + i * P);
        }
        op += step;
    }
    // The groups' sums to shared memory, where the rings were, and from there added in their order.  Their
    // columns differ where their rows' offsets do.
    pdl_trigger();
    float* sw = reinterpret_cast<float*>(ring);   // [R][2][N]
    copy_wait<0>();
    __syncthreads();
    float* mine = sw + threadIdx.x / NT * 2 * N;
#pragma unroll
    for (int i = 0; i < VPT; i++)
#pragma unroll
        for (int j = 0; j < P; j++) {
            float e[2], f[2];
            get(aw[i * P + j], e);
            get(ab[i * P + j], f);
#pragma unroll
            for (int o = 0; o < 2; o++)
                if (cols.has(i, 2 * j + o)) {
                    mine[cols.col(i) + 2 * j + o] = e[o];
                    mine[N + cols.col(i) + 2 * j + o] = f[o];
                }
        }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * N; c += CTA) {
        float v = sw[c];
#pragma unroll
        for (int g = 1; g < R; g++) v += sw[g * 2 * N + c];
        out.put(blockIdx.x, gridDim.x, c, v);
    }
}

// Any row: dx by one CTA, its vectors in registers (K > 0) or in two passes.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kWide) ln_bwd_wide_dx_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                               const T* __restrict__ w, const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, T* __restrict__ dx,
                                                               int64_t N) {
    __shared__ float2 red[32];
    const int64_t base = (int64_t)blockIdx.x * N;
    const float mu = mean[blockIdx.x], rs = rstd[blockIdx.x], inv = 1.f / (float)N;
    RowVec<T, V> xv[K ? K : 1], gv[K ? K : 1];
    auto load = [&](int i, int64_t c) {
        xv[i].load(x + base + c);
        gv[i].load(dy + base + c);
    };
    if (K) each_vector<T, V, K>(N, load);   // all in flight
    float2 s = make_float2(0.f, 0.f);
    each_vector<T, V, K>(N, [&](int i, int64_t c) {
        RowVec<T, V> wv;
        if (!K) load(0, c);
        wv.load(w + c);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float a = gv[i].get(j) * wv.get(j);
            s.x += a;
            s.y += a * ((xv[i].get(j) - mu) * rs);
        }
    });
    s = group_sum2<kWide, 1>(s.x, s.y, red);
    const float c1 = s.x * inv, c2 = s.y * inv;
    each_vector<T, V, K>(N, [&](int i, int64_t c) {
        RowVec<T, V> wv;
        if (!K) load(0, c);
        wv.load(w + c);
        float o[V];
#pragma unroll
        for (int j = 0; j < V; j++) o[j] = rs * (gv[i].get(j) * wv.get(j) - c1 - (xv[i].get(j) - mu) * rs * c2);
        RowVec<T, V>::store(dx + base + c, o);
    });
}

// Any rows: dw and db over the rows of split blockIdx.y, V columns a thread.
template <typename T, int V>
__global__ void __launch_bounds__(256) ln_bwd_wide_cols_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                               const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, const Sums out, int64_t M,
                                                               int64_t N, int64_t rows) {
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= N) return;
    const int64_t r0 = (int64_t)blockIdx.y * rows, r1 = r0 + rows < M ? r0 + rows : M;
    float aw[V], ab[V];
#pragma unroll
    for (int j = 0; j < V; j++) aw[j] = ab[j] = 0.f;
    for (int64_t r = r0; r < r1; r += 4) {   // four rows in flight
        RowVec<T, V> xv[4], gv[4];
        float mu[4], rs[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            xv[k].zero();
            gv[k].zero();
            mu[k] = rs[k] = 0.f;
            if (r + k < r1) {
                xv[k].load(x + (r + k) * N + c);
                gv[k].load(dy + (r + k) * N + c);
                mu[k] = mean[r + k];
                rs[k] = rstd[r + k];
            }
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                aw[j] += gv[k].get(j) * ((xv[k].get(j) - mu[k]) * rs[k]);
                ab[j] += gv[k].get(j);
            }
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        out.put(blockIdx.y, gridDim.y, c + j, aw[j]);
        out.put(blockIdx.y, gridDim.y, N + c + j, ab[j]);
    }
}

// dw[n] (+)= sum_g part[g][0][n], db[n] (+)= sum_g part[g][1][n].  32 columns by
// 32 lanes of rows a CTA, a lane's loads (5 for 148 rows) in flight together; the
// lanes' sums are added in a fixed tree.
__global__ void __launch_bounds__(1024) ln_bwd_final_kernel(const float* __restrict__ part, float* __restrict__ dw,
                                                            float* __restrict__ db, int64_t N, int G, int accumulate) {
    __shared__ float red[32][33];
    pdl_wait();
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float s = 0.f;
    if (c < 2 * N)
        for (int g0 = threadIdx.y; g0 < G; g0 += 32 * 5) {
            float v[5];
#pragma unroll
            for (int k = 0; k < 5; k++) v[k] = g0 + 32 * k < G ? part[(int64_t)(g0 + 32 * k) * 2 * N + c] : 0.f;
#pragma unroll
            for (int k = 0; k < 5; k++) s += v[k];
        }
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = warp_sum(red[threadIdx.x][threadIdx.y]);   // the warp of column threadIdx.y
    const int64_t col = (int64_t)blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x || col >= 2 * N) return;
    float* out = col < N ? dw + col : db + (col - N);
    *out = accumulate ? *out + s : s;
}

// ------------------------------------------------------------------- host --
// Threads of a row's group: 16 elements each, a warp up to 512 elements.
int group_of(int64_t N, int esz) {
    const int V = 16 / esz;
    const int64_t most = N + (N % V ? V - 1 : 0);   // with the largest offset
    for (int threads : {32, 64, 128, 192, 256, 384})
        if (most <= threads * 16) return threads;
    return 512;
}

// Whether the one-pass kernels take a shape (their tensors at 16 bytes).
bool one_pass(int64_t N, int esz) {
    const int V = 16 / esz;
    return N + (N % V ? V - 1 : 0) <= kLnMaxCols;
}

// CTAs for M rows, `rows` of them a CTA at a time and `ctas` to an SM: a number whose stride keeps the rows' offsets
// (their period divides V), or one for each row.
int64_t ctas_for(int64_t M, int64_t N, int esz, int rows, int ctas) {
    const int V = 16 / esz;
    int64_t want = (int64_t)kLnSms * ctas;
    while (N % V && want * rows % V) want--;
    return std::min(want, (M + rows - 1) / rows);
}
// 768 threads an SM, 1024 where a CTA has 512: fewer leave HBM idle, more wait for shared memory and for one another
// (16384 x 2048 bf16 with 512 / 768 / 1024 / 1536: 24.4 / 22.1 / 25.6 / 24.1 us; 4096 x 8192 f32: 62 / 62 / 50 / 60).
int fwd_ctas(int threads) { return (threads == 512 ? 1024 : 768) / threads; }
// CTAs of the backward: an SM's each; one alone, which writes the results itself, for up to two rows a group: as fast
// (8 rows of 2048 bf16 7.1 us, 9 in several CTAs 7.1), with a launch and a workspace less for the host.  More rows a
// group take a microsecond each (8 of them, 128 x 256 f32: 12.6 us, in several CTAs 5.6).
int bwd_rows(int64_t N, int esz) {
    const int nt = group_of(N, esz);
    return (nt % 3 ? 512 : 384) / nt;
}
bool bwd_alone(int64_t M, int64_t N, int esz) {
    const int rows = bwd_rows(N, esz), V = 16 / esz;
    if (!one_pass(N, esz) || M > 2 * rows) return false;
    return N % V == 0 || rows % V == 0 || M <= rows;   // the stride keeps the rows' offsets, or there is none
}
int64_t bwd_ctas(int64_t M, int64_t N, int esz) {
    return bwd_alone(M, N, esz) ? 1 : ctas_for(M, N, esz, bwd_rows(N, esz), 1);
}

// Rows of partial sums that the several-pass backward writes: some six CTAs an SM over tiles of 2048 columns, 16
// rows a split at least.
int64_t wide_parts(int64_t M, int64_t N, int esz) {
    if (bwd_alone(M, N, esz)) return 1;   // the workspace is asked for without the addresses
    const int64_t tiles = (N + 2047) / 2048;
    return std::max<int64_t>(1, std::min((6 * kLnSms + tiles - 1) / tiles, (M + 15) / 16));
}

template <typename T>
int fwd(tb_ctx* ctx, const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, int64_t M, int64_t N, float eps) {
    constexpr int V = 16 / sizeof(T);
    if (!one_pass(N, sizeof(T)) || !aligned16(x) || !aligned16(y)) {
        const bool vec = N % V == 0 && aligned16(x) && aligned16(y) && aligned16(w) && aligned16(b);
        constexpr int K = 16 / V;   // rows of up to 16384 in registers
        auto kern = !vec ? ln_fwd_wide_kernel<T, 1, 0> : N <= kWide * 16 ? ln_fwd_wide_kernel<T, V, K> : ln_fwd_wide_kernel<T, V, 0>;
        return launch(ctx, "layernorm_fwd_wide", kern, dim3((unsigned)M), dim3(kWide), 0, x, w, b, y, mean, rstd, N, eps);
    }
    const int nt = group_of(N, sizeof(T)), threads = nt == 32 ? 256 : nt;
    const int64_t grid = ctas_for(M, N, sizeof(T), threads / nt, fwd_ctas(threads));
    const int smem = kLnStages * threads * 16 * (int)sizeof(T);
    auto go = [&](auto kern) {
        if (smem > 47 * 1024)   // with the static part, past what a kernel has unasked
            TB_CUDA_TRY(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        return launch(ctx, "layernorm_fwd", kern, dim3((unsigned)grid), dim3(threads), smem, x, w, b, y, mean, rstd, M,
                      (int)N, eps);
    };
    auto of = [&](auto shift) {
        constexpr bool SH = decltype(shift)::value;
        constexpr int K = 16 / V;
        switch (nt) {
            case 32: return go(ln_fwd_kernel<T, K, 32, SH>);
            case 64: return go(ln_fwd_kernel<T, K, 64, SH>);
            case 128: return go(ln_fwd_kernel<T, K, 128, SH>);
            case 192: return go(ln_fwd_kernel<T, K, 192, SH>);
            case 256: return go(ln_fwd_kernel<T, K, 256, SH>);
            case 384: return go(ln_fwd_kernel<T, K, 384, SH>);
            default: return go(ln_fwd_kernel<T, K, 512, SH>);
        }
    };
    return N % V ? of(std::true_type()) : of(std::false_type());
}

template <typename T>
int bwd(tb_ctx* ctx, const T* dy, const T* x, const T* w, const float* mean, const float* rstd, T* dx, float* dw, float* db,
        int accumulate, int64_t M, int64_t N, float* part) {
    constexpr int V = 16 / sizeof(T);
    const Sums out = {part, dw, db, N, accumulate};
    int64_t G;
    int rc;
    if (!one_pass(N, sizeof(T)) || !aligned16(x) || !aligned16(dy) || !aligned16(dx)) {
        const bool vec = N % V == 0 && aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(w);
        const int cols = 256 * (vec ? V : 1);
        G = wide_parts(M, N, sizeof(T));
        constexpr int K = 16 / V;   // rows of up to 16384 in registers
        auto kern = !vec ? ln_bwd_wide_dx_kernel<T, 1, 0> : N <= kWide * 16 ? ln_bwd_wide_dx_kernel<T, V, K> : ln_bwd_wide_dx_kernel<T, V, 0>;
        rc = launch(ctx, "layernorm_bwd_wide", kern, dim3((unsigned)M), dim3(kWide), 0, dy, x, w, mean, rstd, dx, N);
        if (rc) return rc;
        rc = launch(ctx, "layernorm_bwd_cols", vec ? ln_bwd_wide_cols_kernel<T, V> : ln_bwd_wide_cols_kernel<T, 1>,
                    dim3((unsigned)((N + cols - 1) / cols), (unsigned)G), dim3(256), 0, dy, x, mean, rstd, out, M, N,
                    (M + G - 1) / G);
    } else {
        const int nt = group_of(N, sizeof(T)), threads = nt % 3 ? 512 : 384;
        G = bwd_ctas(M, N, sizeof(T));
        const int smem = kLnStages * 2 * threads * 16 * (int)sizeof(T);   // the groups' sums take 8 N bytes each, 64 KB at most
        auto go = [&](auto kern) {
            TB_CUDA_TRY(ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            return launch(ctx, "layernorm_bwd", kern, dim3((unsigned)G), dim3(threads), smem, dy, x, w, mean, rstd, dx, out,
                          M, (int)N);
        };
        auto of = [&](auto shift) {
            constexpr bool SH = decltype(shift)::value;
            constexpr int K = 16 / V;
            switch (nt) {
                case 32: return go(ln_bwd_kernel<T, K, 32, SH>);
                case 64: return go(ln_bwd_kernel<T, K, 64, SH>);
                case 128: return go(ln_bwd_kernel<T, K, 128, SH>);
                case 192: return go(ln_bwd_kernel<T, K, 192, SH>);
                case 256: return go(ln_bwd_kernel<T, K, 256, SH>);
                case 384: return go(ln_bwd_kernel<T, K, 384, SH>);
                default: return go(ln_bwd_kernel<T, K, 512, SH>);
            }
        };
        rc = N % V ? of(std::true_type()) : of(std::false_type());
    }
    if (rc || G == 1) return rc;
    // launched while the last CTAs still run: it waits for them itself
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)((2 * N + 31) / 32));
    lc.blockDim = dim3(32, 32);
    lc.stream = ctx->stream;
    cudaLaunchAttribute early[1];
    early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = early;
    lc.numAttrs = 1;
    TB_CUDA_TRY(ctx, cudaLaunchKernelEx(&lc, ln_bwd_final_kernel, (const float*)part, dw, db, N, (int)G, accumulate));
    return TB_OK;
}

struct Span {
    const void* p;
    size_t bytes;
};
// Whether one of the first `outs` spans meets another span.
bool meet(const Span* s, int n, int outs) {
    for (int i = 0; i < outs; i++)
        for (int j = i + 1; j < n; j++) {
            const uintptr_t a = (uintptr_t)s[i].p, b = (uintptr_t)s[j].p;
            if (a < b + s[j].bytes && b < a + s[i].bytes) return true;
        }
    return false;
}
bool aligned_to(size_t a, std::initializer_list<const void*> ps) {
    for (const void* p : ps)
        if ((uintptr_t)p & (a - 1)) return false;
    return true;
}

bool ln_shape_ok(int64_t M, int64_t N) {
    // rows index a grid, and no offset passes 64 bits
    return M >= 0 && N > 0 && M < (1ll << 31) && N < (1ll << 31);
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" {

int tb_layernorm_fwd_train(tb_ctx* ctx, int dtype, const void* x, const void* w, const void* b, void* y, float* mean,
                           float* rstd, int64_t M, int64_t N, float eps) {
    if (!ctx) return TB_ERR_ARG;
    if (dtype != TB_F32 && dtype != TB_BF16)
        return set_error(ctx, TB_ERR_UNSUPPORTED, "layernorm_fwd_train: dtype %d", dtype);
    TB_REQUIRE(ctx, ln_shape_ok(M, N), TB_ERR_SHAPE, "layernorm_fwd_train: M=%lld N=%lld", (long long)M, (long long)N);
    if (M == 0) return TB_OK;
    TB_REQUIRE(ctx, x && w && b && y && mean && rstd, TB_ERR_ARG, "layernorm_fwd_train: null pointer");
    const size_t es = dtype == TB_F32 ? 4 : 2, row = es * (size_t)N, all = row * (size_t)M;
    TB_REQUIRE(ctx, aligned_to(es, {x, w, b, y}) && aligned_to(4, {mean, rstd}), TB_ERR_ALIGN,
               "layernorm_fwd_train: a pointer is not aligned to its type");
    const size_t stat = 4 * (size_t)M;
    const Span spans[] = {{y, all}, {mean, stat}, {rstd, stat}, {x, all}, {w, row}, {b, row}};
    TB_REQUIRE(ctx, !meet(spans, 6, 3), TB_ERR_ARG, "layernorm_fwd_train: an output overlaps another tensor");
    if (dtype == TB_F32)
        return fwd(ctx, (const float*)x, (const float*)w, (const float*)b, (float*)y, mean, rstd, M, N, eps);
    return fwd(ctx, (const bf16*)x, (const bf16*)w, (const bf16*)b, (bf16*)y, mean, rstd, M, N, eps);
}

int tb_layernorm_bwd(tb_ctx* ctx, int dtype, const void* dy, const void* x, const void* w, const float* mean,
                     const float* rstd, void* dx, float* dw, float* db, int accumulate, int64_t M, int64_t N,
                     void* workspace, size_t workspace_bytes) {
    if (!ctx) return TB_ERR_ARG;
    if (dtype != TB_F32 && dtype != TB_BF16) return set_error(ctx, TB_ERR_UNSUPPORTED, "layernorm_bwd: dtype %d", dtype);
    TB_REQUIRE(ctx, ln_shape_ok(M, N), TB_ERR_SHAPE, "layernorm_bwd: M=%lld N=%lld", (long long)M, (long long)N);
    TB_REQUIRE(ctx, dw && db, TB_ERR_ARG, "layernorm_bwd: null pointer");
    if (M == 0) {   // sums over no rows
        if (!accumulate) {
            TB_CUDA_TRY(ctx, cudaMemsetAsync(dw, 0, (size_t)N * 4, ctx->stream));
            TB_CUDA_TRY(ctx, cudaMemsetAsync(db, 0, (size_t)N * 4, ctx->stream));
        }
        return TB_OK;
    }
    TB_REQUIRE(ctx, dy && x && w && mean && rstd && dx, TB_ERR_ARG, "layernorm_bwd: null pointer");
    const size_t need = tb_layernorm_bwd_ws(dtype, M, N);
    TB_REQUIRE(ctx, !need || (workspace && workspace_bytes >= need), TB_ERR_ARG,
               "layernorm_bwd: workspace of %zu bytes required (tb_workspace_bytes)", need);
    TB_REQUIRE(ctx, aligned16(workspace), TB_ERR_ALIGN, "layernorm_bwd: workspace must be 16-byte aligned");
    const size_t es = dtype == TB_F32 ? 4 : 2, row = es * (size_t)N, all = row * (size_t)M, sums = 4 * (size_t)N;
    TB_REQUIRE(ctx, aligned_to(es, {dy, x, w, dx}) && aligned_to(4, {mean, rstd, dw, db}), TB_ERR_ALIGN,
               "layernorm_bwd: a pointer is not aligned to its type");
    const size_t stat = 4 * (size_t)M;
    const Span spans[] = {{dx, all}, {dw, sums},   {db, sums},   {workspace, need}, {dy, all},
                          {x, all},  {w, row},     {mean, stat}, {rstd, stat}};
    TB_REQUIRE(ctx, !meet(spans, 9, 4), TB_ERR_ARG, "layernorm_bwd: an output overlaps another tensor");
    float* part = reinterpret_cast<float*>(workspace);
    if (dtype == TB_F32)
        return bwd(ctx, (const float*)dy, (const float*)x, (const float*)w, mean, rstd, (float*)dx, dw, db, accumulate, M, N,
                   part);
    return bwd(ctx, (const bf16*)dy, (const bf16*)x, (const bf16*)w, mean, rstd, (bf16*)dx, dw, db, accumulate, M, N, part);
}

size_t tb_layernorm_bwd_ws(int dtype, int64_t M, int64_t N) {
    if (!ln_shape_ok(M, N) || !M) return 0;
    const int esz = dtype == TB_F32 ? 4 : 2;
    // enough for either kernel
    int64_t parts = wide_parts(M, N, esz);
    if (one_pass(N, esz)) parts = std::max(parts, bwd_ctas(M, N, esz));
    return parts > 1 ? (size_t)parts * 2 * (size_t)N * 4 : 0;
}

}  // extern "C"
