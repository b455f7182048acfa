// LayerNorm for training: the forward that keeps each row's mean and rstd, and
// the backward with the reduction of the weight's and the bias's gradients
// (the reference's layer_norm_forward, nn/norm/layernorm.rs:163).
//
//   y = xhat w + b,  xhat = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)
//   a = dy w,  c1 = sum_n(a) / N,  c2 = sum_n(a xhat) / N
//   dx = rstd (a - c1 - xhat c2),  dw = sum_m dy xhat,  db = sum_m dy
//
// Bound by HBM: the forward moves x and y, the backward x, dy and dx, once
// each.  A row lives in the registers of a group of TPR threads (a warp, or the
// CTA), EPT elements a thread, so the mean, the centred variance and the output
// come from one read; the groups walk the rows with the grid's stride and keep w
// (and b) in registers.  In the backward each thread also keeps the f32 sums of
// dw and db for its columns over all the rows it walks; the CTAs write them as
// partial rows, and a second launch adds those in CTA order: no atomics, the
// same bits on each run.  Rows longer than the registers hold take the kernels
// that read a row more than once.
#include <math.h>

#include "rowvec.cuh"

namespace tb {
namespace {

using bf16 = __nv_bfloat16;

// Columns a register kernel holds at most: 1024 threads of 8 elements.
constexpr int64_t kLnMaxCols = 8192;
// CTAs of the backward at most, so that the workspace is a function of the
// shape: 1024 threads an SM on 148 SMs, in CTAs of 256 at least.
constexpr int kLnSms = 148;

__device__ __forceinline__ float2 warp_sum2(float2 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
}

// Sum over a group of TPR threads; groups of more than a warp are the whole CTA
// and go through `red` (TPR / 32 entries).  The caller alternates two buffers:
// a thread that writes one again has passed the barrier of the other, which
// every reader of the first has reached.
template <int TPR>
__device__ __forceinline__ float2 group_sum2(float2 v, float2* red) {
    v = warp_sum2(v);
    if (TPR == 32) return v;
    constexpr int W = TPR / 32;
    const int lane = threadIdx.x & 31;
    if (lane == 0) red[threadIdx.x / 32] = v;
    __syncthreads();
    v = red[lane & (W - 1)];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    return v;
}

template <int TPR>
__device__ __forceinline__ float group_sum(float v, float2* red) {
    return group_sum2<TPR>(make_float2(v, 0.f), red).x;
}

// ---------------------------------------------------------------- forward --
template <typename T, int V, int TPR, int EPT>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) ln_fwd_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                                       const T* __restrict__ b, T* __restrict__ y,
                                                                       float* __restrict__ mean, float* __restrict__ rstd,
                                                                       int64_t M, int N, float eps) {
    constexpr int VPT = EPT / V, R = TPR == 32 ? 8 : 1;
    __shared__ float2 red[2][TPR / 32];
    const int t = threadIdx.x % TPR;
    RowVec<T, V> wv[VPT], bv[VPT], xv[VPT];
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int c = (i * TPR + t) * V;
        if (c < N) {
            wv[i].load(w + c);
            bv[i].load(b + c);
        }
    }
    const float inv = 1.f / (float)N;
    for (int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / TPR; row < M; row += (int64_t)gridDim.x * R) {
        const T* xr = x + row * N;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int c = (i * TPR + t) * V;
            if (c < N) xv[i].load(xr + c);
            else xv[i].zero();
#pragma unroll
            for (int j = 0; j < V; j++) s += xv[i].get(j);
        }
        const float mu = group_sum<TPR>(s, red[0]) * inv;
        float q = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; i++)
            if ((i * TPR + t) * V < N)
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float d = xv[i].get(j) - mu;
                    q += d * d;
                }
        const float rs = rsqrtf(group_sum<TPR>(q, red[1]) * inv + eps);
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int c = (i * TPR + t) * V;
            if (c < N) {
                float o[V];
#pragma unroll
                for (int j = 0; j < V; j++) o[j] = (xv[i].get(j) - mu) * rs * wv[i].get(j) + bv[i].get(j);
                RowVec<T, V>::store(y + row * N + c, o);
            }
        }
        if (t == 0) {
            mean[row] = mu;
            rstd[row] = rs;
        }
    }
}

// Rows longer than kLnMaxCols: one CTA a row, three passes (the second and
// third find the row in L2).
template <typename T, int V>
__global__ void __launch_bounds__(1024) ln_fwd_wide_kernel(const T* __restrict__ x, const T* __restrict__ w,
                                                           const T* __restrict__ b, T* __restrict__ y,
                                                           float* __restrict__ mean, float* __restrict__ rstd, int64_t N,
                                                           float eps) {
    __shared__ float2 red[2][32];
    const T* xr = x + (int64_t)blockIdx.x * N;
    T* yr = y + (int64_t)blockIdx.x * N;
    const float inv = 1.f / (float)N;
    RowVec<T, V> v, g, h;
    float s = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < N; c += 1024 * V) {
        v.load(xr + c);
#pragma unroll
        for (int j = 0; j < V; j++) s += v.get(j);
    }
    const float mu = group_sum<1024>(s, red[0]) * inv;
    float q = 0.f;
    for (int64_t c = (int64_t)threadIdx.x * V; c < N; c += 1024 * V) {
        v.load(xr + c);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float d = v.get(j) - mu;
            q += d * d;
        }
    }
    const float rs = rsqrtf(group_sum<1024>(q, red[1]) * inv + eps);
    for (int64_t c = (int64_t)threadIdx.x * V; c < N; c += 1024 * V) {
        v.load(xr + c);
        g.load(w + c);
        h.load(b + c);
        float o[V];
#pragma unroll
        for (int j = 0; j < V; j++) o[j] = (v.get(j) - mu) * rs * g.get(j) + h.get(j);
        RowVec<T, V>::store(yr + c, o);
    }
    if (threadIdx.x == 0) {
        mean[blockIdx.x] = mu;
        rstd[blockIdx.x] = rs;
    }
}

// --------------------------------------------------------------- backward --
// part: [gridDim.x][2][N], the CTA's sums of dw and db.
template <typename T, int V, int TPR, int EPT>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) ln_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                       const T* __restrict__ w,
                                                                       const float* __restrict__ mean,
                                                                       const float* __restrict__ rstd, T* __restrict__ dx,
                                                                       float* __restrict__ part, int64_t M, int N) {
    constexpr int VPT = EPT / V, R = TPR == 32 ? 8 : 1;
    __shared__ float2 red[2][TPR / 32];
    const int t = threadIdx.x % TPR;
    RowVec<T, V> wv[VPT], xv[VPT], gv[VPT];
    float aw[EPT], ab[EPT];
#pragma unroll
    for (int i = 0; i < VPT; i++) {
        const int c = (i * TPR + t) * V;
        if (c < N) wv[i].load(w + c);
        else wv[i].zero();
#pragma unroll
        for (int j = 0; j < V; j++) aw[i * V + j] = ab[i * V + j] = 0.f;
    }
    const float inv = 1.f / (float)N;
    int buf = 0;
    for (int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / TPR; row < M; row += (int64_t)gridDim.x * R) {
        const float mu = mean[row], rs = rstd[row];
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int c = (i * TPR + t) * V;
            if (c < N) {
                xv[i].load(x + row * N + c);
                gv[i].load(dy + row * N + c);
            } else {
                xv[i].zero();
                gv[i].zero();
            }
        }
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < VPT; i++)
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float g = gv[i].get(j), xh = (xv[i].get(j) - mu) * rs, a = g * wv[i].get(j);
                s.x += a;
                s.y += a * xh;
                aw[i * V + j] += g * xh;
                ab[i * V + j] += g;
            }
        s = group_sum2<TPR>(s, red[buf]);
        buf ^= 1;
        const float c1 = s.x * inv, c2 = s.y * inv;
#pragma unroll
        for (int i = 0; i < VPT; i++) {
            const int c = (i * TPR + t) * V;
            if (c < N) {
                float o[V];
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float xh = (xv[i].get(j) - mu) * rs;
                    o[j] = rs * (gv[i].get(j) * wv[i].get(j) - c1 - xh * c2);
                }
                RowVec<T, V>::store(dx + row * N + c, o);
            }
        }
    }
    if (R > 1) {   // the warps' sums, added in warp order
        __shared__ float sw[R > 1 ? 32 * EPT : 1], sb[R > 1 ? 32 * EPT : 1];
        for (int r = 0; r < R; r++) {
            if (threadIdx.x / 32 == r)
#pragma unroll
                for (int k = 0; k < EPT; k++) {
                    const int c = k * 32 + t;
                    if (r) {
                        aw[k] += sw[c];
                        ab[k] += sb[c];
                    }
                    sw[c] = aw[k];
                    sb[c] = ab[k];
                }
            __syncthreads();
        }
        if (threadIdx.x / 32 != R - 1) return;
    }
    float* pw = part + (int64_t)blockIdx.x * 2 * N;
#pragma unroll
    for (int i = 0; i < VPT; i++)
#pragma unroll
        for (int j = 0; j < V; j++) {
            const int c = (i * TPR + t) * V + j;
            if (c < N) {
                pw[c] = aw[i * V + j];
                pw[N + c] = ab[i * V + j];
            }
        }
}

// Long rows: dx by one CTA a row, two passes.
template <typename T, int V>
__global__ void __launch_bounds__(1024) ln_bwd_wide_dx_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                              const T* __restrict__ w, const float* __restrict__ mean,
                                                              const float* __restrict__ rstd, T* __restrict__ dx,
                                                              int64_t N) {
    __shared__ float2 red[32];
    const int64_t base = (int64_t)blockIdx.x * N;
    const float mu = mean[blockIdx.x], rs = rstd[blockIdx.x], inv = 1.f / (float)N;
    RowVec<T, V> xv, gv, wv;
    float2 s = make_float2(0.f, 0.f);
    for (int64_t c = (int64_t)threadIdx.x * V; c < N; c += 1024 * V) {
        xv.load(x + base + c);
        gv.load(dy + base + c);
        wv.load(w + c);
#pragma unroll
        for (int j = 0; j < V; j++) {
            const float a = gv.get(j) * wv.get(j);
            s.x += a;
            s.y += a * ((xv.get(j) - mu) * rs);
        }
    }
    s = group_sum2<1024>(s, red);
    const float c1 = s.x * inv, c2 = s.y * inv;
    for (int64_t c = (int64_t)threadIdx.x * V; c < N; c += 1024 * V) {
        xv.load(x + base + c);
        gv.load(dy + base + c);
        wv.load(w + c);
        float o[V];
#pragma unroll
        for (int j = 0; j < V; j++)
            o[j] = rs * (gv.get(j) * wv.get(j) - c1 - (xv.get(j) - mu) * rs * c2);
        RowVec<T, V>::store(dx + base + c, o);
    }
}

// Long rows: dw and db over the rows of split blockIdx.y, V columns a thread.
template <typename T, int V>
__global__ void __launch_bounds__(256) ln_bwd_wide_cols_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                               const float* __restrict__ mean,
                                                               const float* __restrict__ rstd, float* __restrict__ part,
                                                               int64_t M, int64_t N, int64_t rows) {
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
    if (c >= N) return;
    const int64_t r0 = (int64_t)blockIdx.y * rows, r1 = r0 + rows < M ? r0 + rows : M;
    float aw[V], ab[V];
#pragma unroll
    for (int j = 0; j < V; j++) aw[j] = ab[j] = 0.f;
    RowVec<T, V> xv, gv;
#pragma unroll 4
    for (int64_t r = r0; r < r1; r++) {
        xv.load(x + r * N + c);
        gv.load(dy + r * N + c);
        const float mu = mean[r], rs = rstd[r];
#pragma unroll
        for (int j = 0; j < V; j++) {
            aw[j] += gv.get(j) * ((xv.get(j) - mu) * rs);
            ab[j] += gv.get(j);
        }
    }
    float* pw = part + (int64_t)blockIdx.y * 2 * N;
#pragma unroll
    for (int j = 0; j < V; j++) {
        pw[c + j] = aw[j];
        pw[N + c + j] = ab[j];
    }
}

// dw[n] (+)= sum_g part[g][0][n], db[n] (+)= sum_g part[g][1][n].  32 columns by
// 16 lanes of rows a CTA; the lanes' sums are added in lane order.
__global__ void __launch_bounds__(512) ln_bwd_final_kernel(const float* __restrict__ part, float* __restrict__ dw,
                                                           float* __restrict__ db, int64_t N, int G, int accumulate) {
    __shared__ float red[16][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float s = 0.f;
    if (c < 2 * N)
#pragma unroll 4
        for (int g = threadIdx.y; g < G; g += 16) s += part[(int64_t)g * 2 * N + c];
    red[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y || c >= 2 * N) return;
#pragma unroll
    for (int k = 1; k < 16; k++) s += red[k][threadIdx.x];
    float* out = c < N ? dw + c : db + (c - N);
    *out = accumulate ? *out + s : s;
}

// ------------------------------------------------------------------- host --
// Threads that share a row, and the rows a CTA takes at a time.
int group_threads(int64_t N) { return N <= 256 ? 32 : N <= 1024 ? 128 : N <= 2048 ? 256 : N <= 4096 ? 512 : 1024; }

// Rows of partial sums that the backward writes.
int64_t bwd_parts(int64_t M, int64_t N) {
    if (N > kLnMaxCols) {
        // two CTAs an SM or so over tiles of at most 2048 columns, 16 rows a split at least
        const int64_t tiles = (N + 2047) / 2048, want = (2 * kLnSms + tiles - 1) / tiles, most = (M + 15) / 16;
        return want < most ? want : most;
    }
    const int tpr = group_threads(N), threads = tpr == 32 ? 256 : tpr, rows = tpr == 32 ? 8 : 1;
    const int64_t want = (int64_t)kLnSms * (1024 / threads), most = (M + rows - 1) / rows;
    return want < most ? want : most;
}

template <typename T, int V>
int fwd(tb_ctx* ctx, const T* x, const T* w, const T* b, T* y, float* mean, float* rstd, int64_t M, int64_t N, float eps) {
    if (N > kLnMaxCols)
        return launch(ctx, "layernorm_fwd_wide", ln_fwd_wide_kernel<T, V>, dim3((unsigned)M), dim3(1024), 0, x, w, b, y,
                      mean, rstd, N, eps);
    const int tpr = group_threads(N), threads = tpr == 32 ? 256 : tpr, rows = tpr == 32 ? 8 : 1;
    const int64_t want = (int64_t)ctx->num_sms * (2048 / threads), most = (M + rows - 1) / rows;
    const dim3 grid((unsigned)(want < most ? want : most));
    auto go = [&](auto kern) {
        return launch(ctx, "layernorm_fwd", kern, grid, dim3(threads), 0, x, w, b, y, mean, rstd, M, (int)N, eps);
    };
    switch (tpr) {
        case 32: return go(ln_fwd_kernel<T, V, 32, 8>);
        case 128: return go(ln_fwd_kernel<T, V, 128, 8>);
        case 256: return go(ln_fwd_kernel<T, V, 256, 8>);
        case 512: return go(ln_fwd_kernel<T, V, 512, 8>);
        default: return go(ln_fwd_kernel<T, V, 1024, 8>);
    }
}

template <typename T, int V>
int bwd(tb_ctx* ctx, const T* dy, const T* x, const T* w, const float* mean, const float* rstd, T* dx, float* dw, float* db,
        int accumulate, int64_t M, int64_t N, float* part) {
    const int64_t G = bwd_parts(M, N);
    int rc;
    if (N > kLnMaxCols) {
        rc = launch(ctx, "layernorm_bwd_wide", ln_bwd_wide_dx_kernel<T, V>, dim3((unsigned)M), dim3(1024), 0, dy, x, w,
                    mean, rstd, dx, N);
        if (rc) return rc;
        const int64_t rows = (M + G - 1) / G;
        rc = launch(ctx, "layernorm_bwd_cols", ln_bwd_wide_cols_kernel<T, V>,
                    dim3((unsigned)((N + 256 * V - 1) / (256 * V)), (unsigned)G), dim3(256), 0, dy, x, mean, rstd, part, M,
                    N, rows);
    } else {
        const int tpr = group_threads(N), threads = tpr == 32 ? 256 : tpr;
        auto go = [&](auto kern) {
            return launch(ctx, "layernorm_bwd", kern, dim3((unsigned)G), dim3(threads), 0, dy, x, w, mean, rstd, dx, part, M,
                          (int)N);
        };
        switch (tpr) {
            case 32: rc = go(ln_bwd_kernel<T, V, 32, 8>); break;
            case 128: rc = go(ln_bwd_kernel<T, V, 128, 8>); break;
            case 256: rc = go(ln_bwd_kernel<T, V, 256, 8>); break;
            case 512: rc = go(ln_bwd_kernel<T, V, 512, 8>); break;
            default: rc = go(ln_bwd_kernel<T, V, 1024, 8>); break;
        }
    }
    if (rc) return rc;
    return launch(ctx, "layernorm_bwd_final", ln_bwd_final_kernel, dim3((unsigned)((2 * N + 31) / 32)), dim3(32, 16), 0,
                  (const float*)part, dw, db, N, (int)G, accumulate);
}

// Whether the bytes at p meet those at q.
bool meet(const void* p, size_t np, const void* q, size_t nq) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    return a < b + nq && b < a + np;
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
    TB_REQUIRE(ctx, !meet(y, all, x, all) && !meet(y, all, w, row) && !meet(y, all, b, row), TB_ERR_ARG,
               "layernorm_fwd_train: y overlaps an input");
    const bool vec = aligned16(x) && aligned16(w) && aligned16(b) && aligned16(y);
    if (dtype == TB_F32) {
        auto f = vec && N % 4 == 0 ? fwd<float, 4> : fwd<float, 1>;
        return f(ctx, (const float*)x, (const float*)w, (const float*)b, (float*)y, mean, rstd, M, N, eps);
    }
    auto f = vec && N % 8 == 0 ? fwd<bf16, 8> : fwd<bf16, 1>;
    return f(ctx, (const bf16*)x, (const bf16*)w, (const bf16*)b, (bf16*)y, mean, rstd, M, N, eps);
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
    const size_t need = tb_layernorm_bwd_ws(M, N);
    TB_REQUIRE(ctx, workspace && workspace_bytes >= need, TB_ERR_ARG,
               "layernorm_bwd: workspace of %zu bytes required (tb_workspace_bytes)", need);
    TB_REQUIRE(ctx, aligned16(workspace), TB_ERR_ALIGN, "layernorm_bwd: workspace must be 16-byte aligned");
    const size_t es = dtype == TB_F32 ? 4 : 2, row = es * (size_t)N, all = row * (size_t)M, sums = 4 * (size_t)N;
    TB_REQUIRE(ctx, !meet(dx, all, x, all) && !meet(dx, all, dy, all) && !meet(dx, all, w, row) && !meet(dw, sums, db, sums),
               TB_ERR_ARG, "layernorm_bwd: an output overlaps another tensor");
    float* part = reinterpret_cast<float*>(workspace);
    const bool vec = aligned16(dy) && aligned16(x) && aligned16(w) && aligned16(dx);
    if (dtype == TB_F32) {
        auto f = vec && N % 4 == 0 ? bwd<float, 4> : bwd<float, 1>;
        return f(ctx, (const float*)dy, (const float*)x, (const float*)w, mean, rstd, (float*)dx, dw, db, accumulate, M, N,
                 part);
    }
    auto f = vec && N % 8 == 0 ? bwd<bf16, 8> : bwd<bf16, 1>;
    return f(ctx, (const bf16*)dy, (const bf16*)x, (const bf16*)w, mean, rstd, (bf16*)dx, dw, db, accumulate, M, N, part);
}

size_t tb_layernorm_bwd_ws(int64_t M, int64_t N) {
    return ln_shape_ok(M, N) ? (size_t)bwd_parts(M, N) * 2 * (size_t)N * 4 : 0;
}

}  // extern "C"
