// qk_norm_rope.cu -- norms of queries and keys for each head with the position rotation in the same pass, and the backward pass.
//
//   xhat = (x - mu) * r,  r = 1 / sqrt(mean((x - mu)^2) + eps)     over one head of one token (mu = 0 for the root mean square)
//   n    = xhat * w
//   y    = n with its first `rot` dims rotated: (a, b) -> (a cos - b sin, b cos + a sin), pairs (i, i + rot / 2) or (2 i, 2 i + 1)
// Backward, from x and dy alone (nothing is kept by the forward pass):
//   g    = dy with the rotation turned back,  dw = sum over tokens and heads of g * xhat,  gh = g * w
//   dx   = r * (gh - mean(gh) - xhat * mean(gh * xhat))            (without the mean(gh) term for the root mean square)
// All of it in fp32, rounded once where a result is stored.  Every pass is bound by the bytes of Q, K and their results.
#include "i8_common.cuh"

namespace ppml_b200 {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

constexpr int kWarps = 8;

// What one row (a head of a token) needs to know.
struct Row { long long t; int b, l, h, pos; bool key, skip, bad; };

__device__ __forceinline__ Row row_of(const QkParams& p, long long r) {
    Row w;
    const int H = p.hq + p.hk;
    w.t = r / H;
    const int h = static_cast<int>(r - w.t * H);
    w.b = static_cast<int>(w.t / p.L);
    w.l = static_cast<int>(w.t - static_cast<long long>(w.b) * p.L);
    w.key = h >= p.hq;
    w.h = w.key ? h - p.hq : h;
    w.pos = p.positions ? p.positions[w.b * p.pos_b + w.l] : w.l;
    w.skip = w.pos < 0;
    w.bad = p.rot > 0 && w.pos >= p.table_rows;
    return w;
}
template <typename T>
__device__ __forceinline__ T* row_ptr(const HeadsView& v, const Row& w) {
    return static_cast<T*>(v.p) + w.b * v.b + w.l * v.l + w.h * v.h;
}

// One warp per row, element lane + 32 i of the row in register i; rotation partners meet in shared memory.
template <typename T, int N>
__global__ void __launch_bounds__(32 * kWarps) qk_forward_kernel(const QkParams p) {
    __shared__ float buf[kWarps][32 * N];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* row = buf[warp];
    const long long rows = static_cast<long long>(p.B) * p.L * (p.hq + p.hk);
    const float inv_d = 1.0f / static_cast<float>(p.d);
    for (long long r = static_cast<long long>(blockIdx.x) * kWarps + warp; r < rows; r += static_cast<long long>(gridDim.x) * kWarps) {
        const Row w = row_of(p, r);
        if (w.skip) continue;
        const T* src = row_ptr<const T>(w.key ? p.k : p.q, w);
        T* dst = row_ptr<T>(w.key ? p.ko : p.qo, w);
        const float* wt = w.key ? p.kw : p.qw;
        float x[N];
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = lane + 32 * i < p.d ? to_f32(src[lane + 32 * i]) : 0.0f;
        if (p.norm == 2) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) s += x[i];
            const float mu = warp_sum(s) * inv_d;
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = lane + 32 * i < p.d ? x[i] - mu : 0.0f;
        }
        float rs = 1.0f;
        if (p.norm != 0) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) s = fmaf(x[i], x[i], s);
            rs = 1.0f / sqrtf(warp_sum(s) * inv_d + p.eps);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] *= rs;
            if (wt && lane + 32 * i < p.d) x[i] *= wt[lane + 32 * i];
        }
        if (p.rot > 0) {
            const int half = p.rot / 2;
#pragma unroll
            for (int i = 0; i < N; ++i) row[lane + 32 * i] = x[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = lane + 32 * i;
                if (e >= p.rot) continue;
                const int j = p.interleaved ? e >> 1 : (e < half ? e : e - half);
                const bool second = p.interleaved ? (e & 1) : e >= half;
                const int o = p.interleaved ? (e ^ 1) : (second ? e - half : e + half);
                const long long at = static_cast<long long>(w.pos) * half + j;
                const float c = w.bad ? __uint_as_float(0x7fffffffu) : p.cos_t[at], s = w.bad ? 0.0f : p.sin_t[at];
                x[i] = second ? fmaf(row[o], s, x[i] * c) : fmaf(-row[o], s, x[i] * c);
            }
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + 32 * i < p.d) dst[lane + 32 * i] = from_f32<T>(x[i]);
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(32 * kWarps) qk_backward_kernel(const QkParams p) {
    __shared__ float buf[kWarps][32 * N];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* row = buf[warp];
    const long long rows = static_cast<long long>(p.B) * p.L * (p.hq + p.hk);
    const float inv_d = 1.0f / static_cast<float>(p.d);
    float dwq[N], dwk[N];
#pragma unroll
    for (int i = 0; i < N; ++i) dwq[i] = dwk[i] = 0.0f;
    for (long long r = static_cast<long long>(blockIdx.x) * kWarps + warp; r < rows; r += static_cast<long long>(gridDim.x) * kWarps) {
        const Row w = row_of(p, r);
        const T* src = row_ptr<const T>(w.key ? p.k : p.q, w);
        const T* dy = row_ptr<const T>(w.key ? p.ko : p.qo, w);
        T* dst = row_ptr<T>(w.key ? p.dk : p.dq, w);
        const float* wt = w.key ? p.kw : p.qw;
        if (w.skip) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (lane + 32 * i < p.d) dst[lane + 32 * i] = from_f32<T>(0.0f);
            continue;
        }
        float x[N], g[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool in = lane + 32 * i < p.d;
            x[i] = in ? to_f32(src[lane + 32 * i]) : 0.0f;
            g[i] = in ? to_f32(dy[lane + 32 * i]) : 0.0f;
        }
        if (p.rot > 0) {
            const int half = p.rot / 2;
#pragma unroll
            for (int i = 0; i < N; ++i) row[lane + 32 * i] = g[i];
            __syncwarp();
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int e = lane + 32 * i;
                if (e >= p.rot) continue;
                const int j = p.interleaved ? e >> 1 : (e < half ? e : e - half);
                const bool second = p.interleaved ? (e & 1) : e >= half;
                const int o = p.interleaved ? (e ^ 1) : (second ? e - half : e + half);
                const long long at = static_cast<long long>(w.pos) * half + j;
                const float c = w.bad ? __uint_as_float(0x7fffffffu) : p.cos_t[at], s = w.bad ? 0.0f : p.sin_t[at];
                g[i] = second ? fmaf(-row[o], s, g[i] * c) : fmaf(row[o], s, g[i] * c);
            }
            __syncwarp();
        }
        float rs = 1.0f;
        if (p.norm == 2) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) s += x[i];
            const float mu = warp_sum(s) * inv_d;
#pragma unroll
            for (int i = 0; i < N; ++i) x[i] = lane + 32 * i < p.d ? x[i] - mu : 0.0f;
        }
        if (p.norm != 0) {
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) s = fmaf(x[i], x[i], s);
            rs = 1.0f / sqrtf(warp_sum(s) * inv_d + p.eps);
        }
        float sg = 0.0f, sgx = 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            x[i] *= rs;
            if (w.key) dwk[i] = fmaf(g[i], x[i], dwk[i]); else dwq[i] = fmaf(g[i], x[i], dwq[i]);
            if (wt && lane + 32 * i < p.d) g[i] *= wt[lane + 32 * i];
            sg += g[i];
            sgx = fmaf(g[i], x[i], sgx);
        }
        if (p.norm != 0) {
            sgx = warp_sum(sgx) * inv_d;
            sg = p.norm == 2 ? warp_sum(sg) * inv_d : 0.0f;
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = rs * (g[i] - sg - x[i] * sgx);
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (lane + 32 * i < p.d) dst[lane + 32 * i] = from_f32<T>(g[i]);
    }
    if (!p.partial) return;
    // the warps of a block in order, one line of the workspace per block
    for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) row[lane + 32 * i] = k ? dwk[i] : dwq[i];
        __syncthreads();
        for (int e = threadIdx.x; e < p.d; e += 32 * kWarps) {
            float s = 0.0f;
            for (int v = 0; v < kWarps; ++v) s += buf[v][e];
            p.partial[(static_cast<long long>(k) * gridDim.x + blockIdx.x) * p.d + e] = s;
        }
    }
}

// dw[e] = sum over the blocks' lines, in order; one warp per element and side
__global__ void __launch_bounds__(128) qk_weight_sum_kernel(const float* __restrict__ partial, int lines, int d, float* dqw, float* dkw) {
    const int e = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31, k = blockIdx.y;
    float* out = k ? dkw : dqw;
    if (e >= d || !out) return;
    float s = 0.0f;
    for (int i = lane; i < lines; i += 32) s += partial[(static_cast<long long>(k) * lines + i) * d + e];
    s = warp_sum(s);
    if (lane == 0) out[e] = s;
}

template <typename T>
int launch_any(const QkParams& p, bool backward, cudaStream_t st) {
    const long long rows = static_cast<long long>(p.B) * p.L * (p.hq + p.hk);
    const unsigned grid = qk_blocks(rows);
    const int n = (p.d + 31) / 32;
#define PPML_QK(N) { if (backward) qk_backward_kernel<T, N><<<grid, 32 * kWarps, 0, st>>>(p); else qk_forward_kernel<T, N><<<grid, 32 * kWarps, 0, st>>>(p); }
    if (n <= 1) PPML_QK(1) else if (n <= 2) PPML_QK(2) else if (n <= 4) PPML_QK(4) else if (n <= 8) PPML_QK(8) else PPML_QK(16)
#undef PPML_QK
    if (cudaGetLastError() != cudaSuccess) return ST_LAUNCH;
    if (backward && p.partial) {
        qk_weight_sum_kernel<<<dim3((p.d + 3) / 4, 2), 128, 0, st>>>(p.partial, static_cast<int>(grid), p.d, p.dqw, p.dkw);
        if (cudaGetLastError() != cudaSuccess) return ST_LAUNCH;
    }
    return ST_OK;
}

}  // namespace

unsigned qk_blocks(long long rows) {
    const long long b = (rows + kWarps - 1) / kWarps;
    return static_cast<unsigned>(b < kQkMaxBlocks ? b : kQkMaxBlocks);
}

int launch_qk_norm_rope(const QkParams& p, int type, bool backward, cudaStream_t st) {
    return type == kTypeF32 ? launch_any<float>(p, backward, st)
                            : type == kTypeF16 ? launch_any<__half>(p, backward, st) : launch_any<__nv_bfloat16>(p, backward, st);
}

}  // namespace ppml_b200
