// qk_norm_rope.cu -- norms of queries and keys for each head with the position rotation in the same pass, and the backward pass.
//
//   xhat = (x - mu) * r,  r = 1 / sqrt(mean((x - mu)^2) + eps)     over one head of one token (mu = 0 for the root mean square)
//   n    = xhat * w
//   y    = n with its first `rot` dims rotated: (a, b) -> (a cos - b sin, b cos + a sin), pairs (i, i + rot / 2) or (2 i, 2 i + 1)
// Backward, from x and dy alone (nothing is kept by the forward pass):
//   g    = dy with the rotation turned back,  dw = sum over tokens and heads of g * xhat,  gh = g * w
//   dx   = r * (gh - mean(gh) - xhat * mean(gh * xhat))            (without the mean(gh) term for the root mean square)
// All of it in fp32, rounded once where a result is stored.  Every pass is bound by the bytes of Q, K and their results.
#include <algorithm>

#include "i8_common.cuh"

namespace ppml_b200 {
namespace {

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The work of a side in the vector kernels: batches of rows per warp, and the steps (tokens, heads) from a batch's row to its next
// and from a warp's batch to its next.
struct QkStep { long long batches, warps; uint32_t jump_t; int jump_h; uint32_t sub_t; int sub_h; };
struct QkVec {
    QkParams p;
    int G;                                         // lanes per row
    unsigned blocks_q;                             // blocks on Q's rows; the others are on K's
    QkStep step_q, step_k;
    uint32_t l_mul; int l_shift;                   // division by L
    int table_vec;                                 // 16-byte reads of the table
};

// ---- any head dim, any alignment: one warp per row ----------------------------------------------------------------------
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


// ---- vector kernels ----------------------------------------------------------------------------------------------------
// A lane holds two chunks of V neighbouring values (VB bytes each) that rotate with one another: chunks l and l + rot / 2 / V for
// the pairs (i, i + rot / 2), chunks 2 l and 2 l + 1 for neighbouring pairs and for dims that pass.  So a rotation needs no
// exchange between lanes, and the table is read once per pair.  G lanes (a power of two) hold a row, a warp W = 32 / G rows.
// A block works on one side (Q or K): its weights stay in registers.  Rows are taken in batches of U * W consecutive ones
// per warp, all of a batch's loads requested before the first is used.
template <int VB> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };

template <typename T, int VB> __device__ __forceinline__ void unpack(const typename RawOf<VB>::type& raw, float* x) {
    constexpr int V = VB / sizeof(T);
    const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = to_f32(t[i]);
}
template <typename T, int VB> __device__ __forceinline__ typename RawOf<VB>::type pack(const float* x) {
    constexpr int V = VB / sizeof(T);
    typename RawOf<VB>::type raw;
    T* t = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = from_f32<T>(x[i]);
    return raw;
}

// n / d for n < 2^31: with 2^s < d <= 2^(s + 1) and m = ceil(2^(32 + s) / d) the error m d - 2^(32 + s) is below 2^(s + 1), so that
// (n m) >> (32 + s) is exact; d = 1 has m = 0.
__device__ __forceinline__ uint32_t div_by(uint32_t n, uint32_t m, int s) { return m == 0 ? n : __umulhi(n, m) >> s; }

struct Side { HeadsView x, y, dx; const float* w; int H; };
__device__ __forceinline__ Side side_of(const QkVec& v, bool key) {
    const QkParams& p = v.p;
    return key ? Side{p.k, p.ko, p.dk, p.kw, p.hk} : Side{p.q, p.qo, p.dq, p.qw, p.hq};
}

// This lane's part of a row and where its pair stands in the table.
template <int V> struct Lane { int a, b, pair; bool has_a, has_b, turns; };
template <int V> __device__ __forceinline__ Lane<V> lane_of(const QkVec& v, int l) {
    Lane<V> n;
    const int chunks = v.p.d / V, half = v.p.interleaved ? 0 : v.p.rot / 2 / V;
    n.turns = v.p.interleaved ? l * V < v.p.rot / 2 : l < half;
    n.a = !v.p.interleaved && l < half ? l : 2 * half + 2 * (l - half);
    n.b = !v.p.interleaved && l < half ? l + half : n.a + 1;
    n.has_a = n.a < chunks; n.has_b = n.b < chunks;
    n.pair = l * V;
    n.a *= V; n.b *= V;
    return n;
}
// cos and sin of the lane's pairs (garbage where none of them turns); NaN beyond the table
template <int V> __device__ __forceinline__ void load_table(const QkVec& v, const Lane<V>& n, int pos, float (&c)[V], float (&s)[V]) {
    const int half = v.p.rot / 2;
#pragma unroll
    for (int i = 0; i < V; ++i) { c[i] = __uint_as_float(0x7fffffffu); s[i] = 0.0f; }
    if (!n.turns || pos >= v.p.table_rows) return;
    const long long at = static_cast<long long>(pos) * half + n.pair;
    if (V % 4 == 0 && v.table_vec) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(v.p.cos_t + at + i);
            *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(v.p.sin_t + at + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (n.pair + i < half) { c[i] = v.p.cos_t[at + i]; s[i] = v.p.sin_t[at + i]; }     // neighbours: may end inside the chunk
    }
}
// x[0 .. V) is the first chunk, x[V .. 2 V) the second; SIGN -1 turns back.  Values that do not turn are not touched: an infinity
// among them must not meet a neighbour, not even times 0.
template <int V, int SIGN> __device__ __forceinline__ void turn(float (&x)[2 * V], const float (&c)[V], const float (&s)[V], const QkParams& p,
                                                                const Lane<V>& n) {
    if (!n.turns) return;
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (n.pair + i >= p.rot / 2) break;
            const float a = x[2 * i], b = x[2 * i + 1];
            x[2 * i] = fmaf(-SIGN * b, s[i], a * c[i]);
            x[2 * i + 1] = fmaf(SIGN * a, s[i], b * c[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float a = x[i], b = x[V + i];
            x[i] = fmaf(-SIGN * b, s[i], a * c[i]);
            x[V + i] = fmaf(SIGN * a, s[i], b * c[i]);
        }
    }
}
__device__ __forceinline__ float group_sum(float v, int G) {
    for (int o = G >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Row t, h of this lane's group and the step to another one.
struct At { uint32_t t; int h; };
__device__ __forceinline__ void advance(At& r, uint32_t dt, int dh, int H) {
    r.t += dt; r.h += dh;
    if (r.h >= H) { r.h -= H; ++r.t; }
}

template <typename T, int VB, int U>
__global__ void __launch_bounds__(256) qk_vec_forward_kernel(const QkVec v) {
    constexpr int V = VB / sizeof(T);
    using Raw = typename RawOf<VB>::type;
    pdl_wait();
    pdl_launch_dependents();
    const bool key = blockIdx.x >= v.blocks_q;
    const Side sd = side_of(v, key);
    const QkStep& st = key ? v.step_k : v.step_q;
    const int lane = threadIdx.x & 31, l = lane & (v.G - 1), g = lane / v.G;
    const Lane<V> n = lane_of<V>(v, l);
    const uint32_t tokens = static_cast<uint32_t>(v.p.B) * static_cast<uint32_t>(v.p.L);
    const float inv_d = 1.0f / static_cast<float>(v.p.d);
    float w[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        w[i] = sd.w && n.has_a ? sd.w[n.a + i] : 1.0f;
        w[V + i] = sd.w && n.has_b ? sd.w[n.b + i] : 1.0f;
    }
    const long long warp = (blockIdx.x - (key ? v.blocks_q : 0u)) * 8ll + (threadIdx.x >> 5);
    const long long r0 = warp * (U * (32 / v.G)) + g;
    At first{static_cast<uint32_t>(min(r0 / sd.H, 0x7fffffffll)), static_cast<int>(r0 % sd.H)};
    for (long long batch = warp; batch < st.batches; batch += st.warps) {
        Raw ra[U], rb[U];
        uint32_t b[U], pl[U]; int h[U], pos[U];
        At r = first;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = r.t < tokens;
            const uint32_t t = in ? r.t : 0u;
            b[u] = div_by(t, v.l_mul, v.l_shift); pl[u] = t - b[u] * static_cast<uint32_t>(v.p.L); h[u] = r.h;
            pos[u] = !in ? -1 : v.p.positions ? v.p.positions[b[u] * v.p.pos_b + pl[u]] : static_cast<int>(pl[u]);
            const T* src = static_cast<const T*>(sd.x.p) + b[u] * sd.x.b + pl[u] * sd.x.l + h[u] * sd.x.h;
            ra[u] = Raw{}; rb[u] = Raw{};
            if (in && n.has_a) ra[u] = *reinterpret_cast<const Raw*>(src + n.a);
            if (in && n.has_b) rb[u] = *reinterpret_cast<const Raw*>(src + n.b);
            advance(r, st.sub_t, st.sub_h, sd.H);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[2 * V], c[V], s[V];
            load_table<V>(v, n, pos[u] < 0 ? 0 : pos[u], c, s);
            unpack<T, VB>(ra[u], x);
            unpack<T, VB>(rb[u], x + V);
            if (v.p.norm == 2) {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) m += x[i];
                m = group_sum(m, v.G) * inv_d;
#pragma unroll
                for (int i = 0; i < V; ++i) { x[i] = n.has_a ? x[i] - m : 0.0f; x[V + i] = n.has_b ? x[V + i] - m : 0.0f; }
            }
            float rs = 1.0f;
            if (v.p.norm != 0) {
                float q = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) q = fmaf(x[i], x[i], q);
                rs = 1.0f / sqrtf(fmaf(group_sum(q, v.G), inv_d, v.p.eps));
            }
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) x[i] = x[i] * rs * w[i];
            turn<V, 1>(x, c, s, v.p, n);
            if (pos[u] >= 0) {
                T* dst = static_cast<T*>(sd.y.p) + b[u] * sd.y.b + pl[u] * sd.y.l + h[u] * sd.y.h;
                if (n.has_a) *reinterpret_cast<Raw*>(dst + n.a) = pack<T, VB>(x);
                if (n.has_b) *reinterpret_cast<Raw*>(dst + n.b) = pack<T, VB>(x + V);
            }
        }
        advance(first, st.jump_t, st.jump_h, sd.H);
    }
}

template <typename T, int VB, int U>
__global__ void __launch_bounds__(256) qk_vec_backward_kernel(const QkVec v) {
    constexpr int V = VB / sizeof(T);
    using Raw = typename RawOf<VB>::type;
    extern __shared__ float sums[];                // [8][d]
    pdl_wait();
    pdl_launch_dependents();
    const bool key = blockIdx.x >= v.blocks_q;
    const Side sd = side_of(v, key);
    const QkStep& st = key ? v.step_k : v.step_q;
    const int lane = threadIdx.x & 31, l = lane & (v.G - 1), g = lane / v.G;
    const Lane<V> n = lane_of<V>(v, l);
    const uint32_t tokens = static_cast<uint32_t>(v.p.B) * static_cast<uint32_t>(v.p.L);
    const float inv_d = 1.0f / static_cast<float>(v.p.d);
    float w[2 * V], dw[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        w[i] = sd.w && n.has_a ? sd.w[n.a + i] : 1.0f;
        w[V + i] = sd.w && n.has_b ? sd.w[n.b + i] : 1.0f;
        dw[i] = dw[V + i] = 0.0f;
    }
    const long long warp = (blockIdx.x - (key ? v.blocks_q : 0u)) * 8ll + (threadIdx.x >> 5);
    const long long r0 = warp * (U * (32 / v.G)) + g;
    At first{static_cast<uint32_t>(min(r0 / sd.H, 0x7fffffffll)), static_cast<int>(r0 % sd.H)};
    for (long long batch = warp; batch < st.batches; batch += st.warps) {
        Raw ra[U], rb[U], ga[U], gb[U];
        uint32_t b[U], pl[U]; int h[U], pos[U]; bool in[U];
        At r = first;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            in[u] = r.t < tokens;
            const uint32_t t = in[u] ? r.t : 0u;
            b[u] = div_by(t, v.l_mul, v.l_shift); pl[u] = t - b[u] * static_cast<uint32_t>(v.p.L); h[u] = r.h;
            pos[u] = !in[u] ? -1 : v.p.positions ? v.p.positions[b[u] * v.p.pos_b + pl[u]] : static_cast<int>(pl[u]);
            const T* src = static_cast<const T*>(sd.x.p) + b[u] * sd.x.b + pl[u] * sd.x.l + h[u] * sd.x.h;
            const T* dy = static_cast<const T*>(sd.y.p) + b[u] * sd.y.b + pl[u] * sd.y.l + h[u] * sd.y.h;
            ra[u] = rb[u] = ga[u] = gb[u] = Raw{};
            if (in[u] && n.has_a) { ra[u] = *reinterpret_cast<const Raw*>(src + n.a); ga[u] = *reinterpret_cast<const Raw*>(dy + n.a); }
            if (in[u] && n.has_b) { rb[u] = *reinterpret_cast<const Raw*>(src + n.b); gb[u] = *reinterpret_cast<const Raw*>(dy + n.b); }
            advance(r, st.sub_t, st.sub_h, sd.H);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float x[2 * V], y[2 * V], c[V], s[V];
            load_table<V>(v, n, pos[u] < 0 ? 0 : pos[u], c, s);
            if (pos[u] < 0) ra[u] = rb[u] = ga[u] = gb[u] = Raw{};             // padding may hold anything: its gradients are 0
            unpack<T, VB>(ra[u], x);
            unpack<T, VB>(rb[u], x + V);
            unpack<T, VB>(ga[u], y);
            unpack<T, VB>(gb[u], y + V);
            turn<V, -1>(y, c, s, v.p, n);
            if (v.p.norm == 2) {
                float m = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) m += x[i];
                m = group_sum(m, v.G) * inv_d;
#pragma unroll
                for (int i = 0; i < V; ++i) { x[i] = n.has_a ? x[i] - m : 0.0f; x[V + i] = n.has_b ? x[V + i] - m : 0.0f; }
            }
            float rs = 1.0f;
            if (v.p.norm != 0) {
                float q = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) q = fmaf(x[i], x[i], q);
                rs = 1.0f / sqrtf(fmaf(group_sum(q, v.G), inv_d, v.p.eps));
            }
            float sg = 0.0f, sgx = 0.0f;
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) {
                x[i] *= rs;
                if (pos[u] >= 0) dw[i] = fmaf(y[i], x[i], dw[i]);              // eps = 0 makes a padded row's xhat NaN
                y[i] *= w[i];
                sg += y[i];
                sgx = fmaf(y[i], x[i], sgx);
            }
            if (v.p.norm != 0) {
                sgx = group_sum(sgx, v.G) * inv_d;
                sg = v.p.norm == 2 ? group_sum(sg, v.G) * inv_d : 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) y[i] = rs * (y[i] - sg - x[i] * sgx);
            }
            if (in[u]) {
                if (pos[u] < 0) {
#pragma unroll
                    for (int i = 0; i < 2 * V; ++i) y[i] = 0.0f;
                }
                T* dst = static_cast<T*>(sd.dx.p) + b[u] * sd.dx.b + pl[u] * sd.dx.l + h[u] * sd.dx.h;
                if (n.has_a) *reinterpret_cast<Raw*>(dst + n.a) = pack<T, VB>(y);
                if (n.has_b) *reinterpret_cast<Raw*>(dst + n.b) = pack<T, VB>(y + V);
            }
        }
        advance(first, st.jump_t, st.jump_h, sd.H);
    }
    if (!v.p.partial) return;
    // the rows of a warp, then the warps of the block in order: one line of the workspace per block
#pragma unroll
    for (int i = 0; i < 2 * V; ++i)
        for (int o = v.G; o < 32; o <<= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
    float* mine = sums + (threadIdx.x >> 5) * v.p.d;
    if (g == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (n.has_a) mine[n.a + i] = dw[i];
            if (n.has_b) mine[n.b + i] = dw[V + i];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < v.p.d; e += 256) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += sums[k * v.p.d + e];
        v.p.partial[static_cast<long long>(blockIdx.x) * v.p.d + e] = s;
    }
}

// dw[e] = sum over a side's lines of the workspace in a fixed order: 32 elements per block, 32 threads on each
__global__ void __launch_bounds__(1024) qk_weight_sum_kernel(const float* __restrict__ partial, int lines_q, int lines_k, int d, float* dqw, float* dkw) {
    __shared__ float part[32][33];
    pdl_wait();
    const bool key = blockIdx.y != 0;
    float* out = key ? dkw : dqw;
    if (!out) return;
    const int e = blockIdx.x * 32 + (threadIdx.x & 31), row = threadIdx.x >> 5;
    const int n = key ? lines_k : lines_q;
    const float* from = partial + (key ? static_cast<long long>(lines_q) * d : 0) + e;
    float s = 0.0f;
    if (e < d) {
#pragma unroll 8
        for (int i = row; i < n; i += 32) s += from[static_cast<long long>(i) * d];
    }
    part[row][threadIdx.x & 31] = s;
    __syncthreads();
    s = warp_sum(part[threadIdx.x & 31][row]);
    if ((threadIdx.x & 31) == 0 && blockIdx.x * 32 + row < d) out[blockIdx.x * 32 + row] = s;
}

// ---- launch ----
unsigned blocks_for(long long rows, int per_block) {
    const long long b = (rows + per_block - 1) / per_block;
    return static_cast<unsigned>(b < kQkMaxBlocks ? b : kQkMaxBlocks);
}

QkStep step_for(long long rows, int H, int per_warp, int W, unsigned blocks) {
    QkStep s{};
    s.batches = (rows + per_warp - 1) / per_warp;
    s.warps = 8ll * blocks;
    const long long jump = s.warps * per_warp;
    s.jump_t = H ? static_cast<uint32_t>(jump / H) : 0; s.jump_h = H ? static_cast<int>(jump % H) : 0;
    s.sub_t = H ? W / H : 0; s.sub_h = H ? W % H : 0;
    return s;
}

template <typename T, int VB, int U>
cudaError_t launch_vec(QkVec& v, bool backward, cudaStream_t st) {
    constexpr int V = VB / sizeof(T);
    const int chunks = v.p.d / V, half = v.p.interleaved ? 0 : v.p.rot / 2 / V;
    const int pairs = half + (chunks - 2 * half + 1) / 2;
    v.G = 1;
    while (v.G < pairs) v.G *= 2;
    const int W = 32 / v.G, per_warp = U * W;
    const long long tokens = static_cast<long long>(v.p.B) * v.p.L, rq = tokens * v.p.hq, rk = tokens * v.p.hk;
    // forward: eight batches a warp at most keep the last wave short; backward: few blocks, as each leaves a line to be summed
    const long long cap = backward ? 2ll * num_sms() : 16ll * num_sms();
    long long bq = (rq + 8 * per_warp - 1) / (8 * per_warp), bk = (rk + 8 * per_warp - 1) / (8 * per_warp);
    if (bq + bk > cap) {
        const long long all = bq + bk;
        bq = bq ? std::max(1ll, cap * bq / all) : 0;
        bk = bk ? std::max(1ll, cap - bq) : 0;
    }
    v.blocks_q = static_cast<unsigned>(bq);
    v.step_q = step_for(rq, v.p.hq, per_warp, W, v.blocks_q);
    v.step_k = step_for(rk, v.p.hk, per_warp, W, static_cast<unsigned>(bk));
    const dim3 grid(static_cast<unsigned>(bq + bk));
    if (!backward) return launch_pdl(qk_vec_forward_kernel<T, VB, U>, grid, dim3(256), 0, st, v);
    cudaError_t e = launch_pdl(qk_vec_backward_kernel<T, VB, U>, grid, dim3(256), v.p.partial ? 8u * v.p.d * sizeof(float) : 0u, st, v);
    if (e == cudaSuccess && v.p.partial)
        e = launch_pdl(qk_weight_sum_kernel, dim3((v.p.d + 31) / 32, 2), dim3(1024), 0, st, static_cast<const float*>(v.p.partial), static_cast<int>(bq),
                       static_cast<int>(bk), v.p.d, v.p.dqw, v.p.dkw);
    return e;
}

// The widest chunk that every base, stride and boundary of the call allows: 16, 8 or 4 bytes, 0 for none.
int chunk_bytes(const QkParams& p, bool backward, int elem) {
    uintptr_t bits = static_cast<uintptr_t>(p.d) * elem;
    if (p.rot > 0 && !p.interleaved) bits |= static_cast<uintptr_t>(p.rot / 2) * elem;
    auto add = [&](const HeadsView& h, int heads) {
        if (heads == 0) return;
        bits |= reinterpret_cast<uintptr_t>(h.p);
        if (p.B > 1) bits |= static_cast<uintptr_t>(h.b) * elem;
        if (p.L > 1) bits |= static_cast<uintptr_t>(h.l) * elem;
        if (heads > 1) bits |= static_cast<uintptr_t>(h.h) * elem;
    };
    add(p.q, p.hq); add(p.k, p.hk); add(p.qo, p.hq); add(p.ko, p.hk);
    if (backward) { add(p.dq, p.hq); add(p.dk, p.hk); }
    for (int vb = 16; vb >= 4; vb /= 2)
        if (bits % vb == 0 && vb >= elem) return p.d * elem <= 64 * vb ? vb : 0;
    return 0;
}

template <typename T>
int launch_any(const QkParams& p, bool backward, cudaStream_t st) {
    QkVec v{};
    v.p = p;
    const int vb = chunk_bytes(p, backward, sizeof(T));
    cudaError_t e;
    if (vb) {
        const uint32_t L = static_cast<uint32_t>(p.L);
        if (L > 1) {
            while ((2u << v.l_shift) < L && v.l_shift < 30) ++v.l_shift;
            v.l_mul = static_cast<uint32_t>(((1ull << (32 + v.l_shift)) + L - 1) / L);
        }
        v.table_vec = (reinterpret_cast<uintptr_t>(p.cos_t) | reinterpret_cast<uintptr_t>(p.sin_t)) % 16 == 0 && (p.rot / 2) % 4 == 0 &&
                      (!p.interleaved || (p.rot / 2) % (vb / sizeof(T)) == 0);
        e = vb == 16 ? launch_vec<T, 16, sizeof(T) == 4 ? 4 : 2>(v, backward, st)
                     : vb == 8 ? launch_vec<T, 8, 4>(v, backward, st) : launch_vec<T, 4, 4>(v, backward, st);
    } else {
        const unsigned grid = blocks_for(static_cast<long long>(p.B) * p.L * (p.hq + p.hk), kWarps);
        const int n = (p.d + 31) / 32;
#define PPML_QK(N) { if (backward) qk_backward_kernel<T, N><<<grid, 32 * kWarps, 0, st>>>(p); else qk_forward_kernel<T, N><<<grid, 32 * kWarps, 0, st>>>(p); }
        if (n <= 1) PPML_QK(1) else if (n <= 2) PPML_QK(2) else if (n <= 4) PPML_QK(4) else if (n <= 8) PPML_QK(8) else PPML_QK(16)
#undef PPML_QK
        e = cudaGetLastError();
        if (e == cudaSuccess && backward && p.partial)
            e = launch_pdl(qk_weight_sum_kernel, dim3((p.d + 31) / 32, 2), dim3(1024), 0, st, static_cast<const float*>(p.partial), static_cast<int>(grid),
                           static_cast<int>(grid), p.d, p.dqw, p.dkw);
    }
    if (e != cudaSuccess) { cudaGetLastError(); return ST_LAUNCH; }
    return ST_OK;
}

}  // namespace

int launch_qk_norm_rope(const QkParams& p, int type, bool backward, cudaStream_t st) {
    return type == kTypeF32 ? launch_any<float>(p, backward, st)
                            : type == kTypeF16 ? launch_any<__half>(p, backward, st) : launch_any<__nv_bfloat16>(p, backward, st);
}

}  // namespace ppml_b200
