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

// What the vector kernels need: byte strides in 32 bits, and how a side's heads are cut into work items.
struct QkView { unsigned char* p; uint32_t b, l, h; };
struct QkSide { QkView x, y, dx; const float* w; int H, per_item, chunks; uint32_t items, blocks, chunks_mul; int chunks_shift; };
struct QkVec {
    QkSide side[2];                                // Q, K
    const float* cos_t; const float* sin_t; const int* positions; float* partial;
    long long pos_b;
    uint32_t L, l_mul; int l_shift;                // division by L
    int d, rot, norm, interleaved, table_rows, table_vec, all_turn;
    int G;                                         // lanes per row
    float eps;
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
// exchange between lanes.  G lanes (a power of two) hold a row, a warp 32 / G of them, of different tokens: each group of
// lanes walks over the heads of its token, so that the position, its table row, the weights and all but one addition of
// an address are had once per token instead of once per row (20 instructions a value before, 6 now).  A block works on one
// side (Q or K).  Where there are few tokens the heads are dealt to several items.
constexpr int kHeadsAtOnce = 4;                    // rows per lane whose loads are in flight together (forward)

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

// 1 / sqrt(v): the hardware's estimate and one Newton step (within 1 unit in the last place; a division and a square root
// take 40 instructions).  0 and infinity stay what the estimate makes of them.
__device__ __forceinline__ float inv_sqrt(float v) {
    const float r = rsqrtf(v);
    return r > 0.0f && r < __uint_as_float(0x7f800000u) ? fmaf(0.5f * r, fmaf(-v * r, r, 1.0f), r) : r;
}

// This lane's part of a row and where its pair stands in the table.
struct Lane { uint32_t a, b; int pair; bool has_a, has_b, turns; };      // a, b: elements
template <int V> __device__ __forceinline__ Lane lane_of(const QkVec& v, int l) {
    Lane n;
    const int chunks = v.d / V, half = v.interleaved ? 0 : v.rot / 2 / V;
    const bool halves = l < half;
    n.turns = v.interleaved ? l * V < v.rot / 2 : halves;
    const int a = halves ? l : 2 * half + 2 * (l - half), b = halves ? l + half : a + 1;
    n.has_a = a < chunks; n.has_b = b < chunks;
    n.pair = l * V;
    n.a = static_cast<uint32_t>(a * V); n.b = static_cast<uint32_t>(b * V);
    return n;
}
// cos and sin of the lane's pairs; NaN beyond the table; 1 and 0 where nothing turns
template <int V> __device__ __forceinline__ void load_table(const QkVec& v, const Lane& n, int pos, float (&c)[V], float (&s)[V]) {
    const int half = v.rot / 2;
    const float none = n.turns && pos >= v.table_rows ? __uint_as_float(0x7fffffffu) : 1.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) { c[i] = n.pair + i < half ? none : 1.0f; s[i] = 0.0f; }
    if (!n.turns || pos >= v.table_rows) return;
    const long long at = static_cast<long long>(pos) * half + n.pair;
    if (V % 4 == 0 && v.table_vec) {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(v.cos_t + at + i);
            *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(v.sin_t + at + i);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (n.pair + i < half) { c[i] = v.cos_t[at + i]; s[i] = v.sin_t[at + i]; }     // neighbours: may end inside the chunk
    }
}
__device__ __forceinline__ float group_sum(float v, int G) {
    for (int o = G >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum over a row, packed pairs of additions inside the lane.
template <int N> __device__ __forceinline__ float lane_sum(const float (&x)[N]) {
    if constexpr (N == 2) return x[0] + x[1];
    uint64_t t = pack2(x[0], x[1]);
#pragma unroll
    for (int i = 2; i < N; i += 2) t = fadd2(t, pack2(x[i], x[i + 1]));
    float a, b; unpack2(t, a, b);
    return a + b;
}
template <int N> __device__ __forceinline__ float lane_dot(const float (&x)[N], const float (&y)[N]) {
    uint64_t t = fmul2(pack2(x[0], x[1]), pack2(y[0], y[1]));
#pragma unroll
    for (int i = 2; i < N; i += 2) t = ffma2(pack2(x[i], x[i + 1]), pack2(y[i], y[i + 1]), t);
    float a, b; unpack2(t, a, b);
    return a + b;
}
// (x - mean) and 1 / sqrt(..) of a row; values that do not exist stay 0
template <int V> __device__ __forceinline__ float normalizer(const QkVec& v, const Lane& n, float inv_d, float (&x)[2 * V]) {
    if (v.norm == 0) return 1.0f;
    if (v.norm == 2) {
        const float m = group_sum(lane_sum(x), v.G) * inv_d;
#pragma unroll
        for (int i = 0; i < V; ++i) { x[i] = n.has_a ? x[i] - m : 0.0f; x[V + i] = n.has_b ? x[V + i] - m : 0.0f; }
    }
    return inv_sqrt(fmaf(group_sum(lane_dot(x, x), v.G), inv_d, v.eps));
}

// The token and heads of an item.
struct Item { int pos, h0, h1; const unsigned char* x; unsigned char* y; unsigned char* dx; };
template <bool BACKWARD> __device__ __forceinline__ Item item_of(const QkVec& v, const QkSide& sd, uint32_t i) {
    Item m{};
    m.pos = -1;
    if (i >= sd.items) return m;
    const uint32_t t = div_by(i, sd.chunks_mul, sd.chunks_shift), chunk = i - t * sd.chunks;
    const uint32_t b = div_by(t, v.l_mul, v.l_shift), l = t - b * v.L;
    m.h0 = static_cast<int>(chunk) * sd.per_item;
    m.h1 = min(m.h0 + sd.per_item, sd.H);
    m.pos = v.positions ? v.positions[static_cast<long long>(b) * v.pos_b + l] : static_cast<int>(l);
    auto at = [&](const QkView& w) {
        return w.p + static_cast<uint64_t>(b) * w.b + static_cast<uint64_t>(l) * w.l + static_cast<uint64_t>(static_cast<uint32_t>(m.h0)) * w.h;
    };
    m.x = at(sd.x); m.y = at(sd.y);
    if (BACKWARD) m.dx = at(sd.dx);
    return m;
}

template <typename T, int VB, int U, int BLOCKS>
__global__ void __launch_bounds__(256, BLOCKS) qk_vec_forward_kernel(const QkVec v) {
    constexpr int V = VB / sizeof(T);
    using Raw = typename RawOf<VB>::type;
    __shared__ float weights[kQkMaxDim + 32];      // a lane past the end of a row reads behind it
    pdl_wait();
    pdl_launch_dependents();
    const bool key = blockIdx.x >= v.side[0].blocks;
    const QkSide& sd = v.side[key];
    const int lane = threadIdx.x & 31, W = 32 / v.G;
    const Lane n = lane_of<V>(v, lane & (v.G - 1));
    const float inv_d = 1.0f / static_cast<float>(v.d);
    const uint32_t warp = (blockIdx.x - (key ? v.side[0].blocks : 0u)) * 8u + (threadIdx.x >> 5), step = sd.blocks * 8u * W;
    for (int e = threadIdx.x; e < kQkMaxDim + 32; e += 256) weights[e] = sd.w && e < v.d ? sd.w[e] : 1.0f;
    __syncthreads();
    for (uint32_t first = warp * W; first < sd.items; first += step) {
        Item m = item_of<false>(v, sd, first + lane / v.G);
        // the result is rs * (x_a (w_a c) - x_b (w_b s), x_b (w_b c) + x_a (w_a s))
        float ac[V], bs[V], bc[V], as[V];
        load_table<V>(v, n, max(m.pos, 0), bc, as);
#pragma unroll
        for (int i = 0; i < V; ++i) {              // neighbours: the lane's two chunks are one run of V pairs
            const float wa = v.interleaved ? weights[n.a + 2 * i] : weights[n.a + i], wb = v.interleaved ? weights[n.a + 2 * i + 1] : weights[n.b + i];
            ac[i] = wa * bc[i]; bs[i] = -wb * as[i]; bc[i] = wb * bc[i]; as[i] = wa * as[i];
        }
        const bool padding = m.pos < 0;
        const int count = m.h1 - m.h0;
        for (int h = 0; h < sd.per_item; h += U) {
            Raw ra[U], rb[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ra[u] = Raw{}; rb[u] = Raw{};
                const T* src = reinterpret_cast<const T*>(m.x + static_cast<uint64_t>(static_cast<uint32_t>(u)) * sd.x.h);
                if (h + u < count && n.has_a) ra[u] = *reinterpret_cast<const Raw*>(src + n.a);
                if (h + u < count && n.has_b) rb[u] = *reinterpret_cast<const Raw*>(src + n.b);
            }
            m.x += static_cast<uint64_t>(U) * sd.x.h;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[2 * V], y[2 * V];
                unpack<T, VB>(ra[u], x);
                unpack<T, VB>(rb[u], x + V);
                const float rs = normalizer<V>(v, n, inv_d, x);
                if (v.interleaved) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float a = x[2 * i] * rs, b = x[2 * i + 1] * rs;
                        y[2 * i] = fmaf(b, bs[i], a * ac[i]);
                        y[2 * i + 1] = fmaf(a, as[i], b * bc[i]);
                    }
                } else if constexpr (V % 2 == 0) {
                    const uint64_t r2 = pack2(rs, rs);
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        const uint64_t a = fmul2(pack2(x[i], x[i + 1]), r2), b = fmul2(pack2(x[V + i], x[V + i + 1]), r2);
                        unpack2(ffma2(b, pack2(bs[i], bs[i + 1]), fmul2(a, pack2(ac[i], ac[i + 1]))), y[i], y[i + 1]);
                        unpack2(ffma2(a, pack2(as[i], as[i + 1]), fmul2(b, pack2(bc[i], bc[i + 1]))), y[V + i], y[V + i + 1]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float a = x[i] * rs, b = x[V + i] * rs;
                        y[i] = fmaf(b, bs[i], a * ac[i]);
                        y[V + i] = fmaf(a, as[i], b * bc[i]);
                    }
                }
                if (!v.all_turn) {                 // dims that pass: an infinity must not meet a neighbour, not even times 0
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        if (n.turns && n.pair + i < v.rot / 2) continue;
                        if (v.interleaved) { y[2 * i] = x[2 * i] * rs * ac[i]; y[2 * i + 1] = x[2 * i + 1] * rs * bc[i]; }
                        else { y[i] = x[i] * rs * ac[i]; y[V + i] = x[V + i] * rs * bc[i]; }
                    }
                }
                if (h + u < count && !padding) {
                    T* dst = reinterpret_cast<T*>(m.y + static_cast<uint64_t>(static_cast<uint32_t>(u)) * sd.y.h);
                    if (n.has_a) *reinterpret_cast<Raw*>(dst + n.a) = pack<T, VB>(y);
                    if (n.has_b) *reinterpret_cast<Raw*>(dst + n.b) = pack<T, VB>(y + V);
                }
            }
            m.y += static_cast<uint64_t>(U) * sd.y.h;
        }
    }
}

template <typename T, int VB, int U, int BLOCKS>
__global__ void __launch_bounds__(256, BLOCKS) qk_vec_backward_kernel(const QkVec v) {
    constexpr int V = VB / sizeof(T);
    using Raw = typename RawOf<VB>::type;
    extern __shared__ float sums[];                // [8][d]
    __shared__ float weights[kQkMaxDim + 32];
    pdl_wait();
    pdl_launch_dependents();
    const bool key = blockIdx.x >= v.side[0].blocks;
    const QkSide& sd = v.side[key];
    const int lane = threadIdx.x & 31, W = 32 / v.G;
    const Lane n = lane_of<V>(v, lane & (v.G - 1));
    const float inv_d = 1.0f / static_cast<float>(v.d);
    const uint32_t warp = (blockIdx.x - (key ? v.side[0].blocks : 0u)) * 8u + (threadIdx.x >> 5), step = sd.blocks * 8u * W;
    for (int e = threadIdx.x; e < kQkMaxDim + 32; e += 256) weights[e] = sd.w && e < v.d ? sd.w[e] : 1.0f;
    __syncthreads();
    float dw[2 * V];
#pragma unroll
    for (int i = 0; i < 2 * V; ++i) dw[i] = 0.0f;
    for (uint32_t first = warp * W; first < sd.items; first += step) {
        Item m = item_of<true>(v, sd, first + lane / v.G);
        float c[V], s[V];
        load_table<V>(v, n, max(m.pos, 0), c, s);
        const bool padding = m.pos < 0;
        const int count = m.h1 - m.h0;
        for (int h = 0; h < sd.per_item; h += U) {
            Raw ra[U], rb[U], ga[U], gb[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ra[u] = rb[u] = ga[u] = gb[u] = Raw{};
                if (h + u >= count || padding) continue;       // padding may hold anything: its gradients are 0
                const T* src = reinterpret_cast<const T*>(m.x + static_cast<uint64_t>(static_cast<uint32_t>(u)) * sd.x.h);
                const T* dy = reinterpret_cast<const T*>(m.y + static_cast<uint64_t>(static_cast<uint32_t>(u)) * sd.y.h);
                if (n.has_a) { ra[u] = *reinterpret_cast<const Raw*>(src + n.a); ga[u] = *reinterpret_cast<const Raw*>(dy + n.a); }
                if (n.has_b) { rb[u] = *reinterpret_cast<const Raw*>(src + n.b); gb[u] = *reinterpret_cast<const Raw*>(dy + n.b); }
            }
            m.x += static_cast<uint64_t>(U) * sd.x.h;
            m.y += static_cast<uint64_t>(U) * sd.y.h;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[2 * V], y[2 * V];
                unpack<T, VB>(ra[u], x);
                unpack<T, VB>(rb[u], x + V);
                unpack<T, VB>(ga[u], y);
                unpack<T, VB>(gb[u], y + V);
                if (n.turns) {
                    if (v.interleaved) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            if (!v.all_turn && n.pair + i >= v.rot / 2) continue;
                            const float a = y[2 * i], b = y[2 * i + 1];
                            y[2 * i] = fmaf(b, s[i], a * c[i]);
                            y[2 * i + 1] = fmaf(-a, s[i], b * c[i]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const float a = y[i], b = y[V + i];
                            y[i] = fmaf(b, s[i], a * c[i]);
                            y[V + i] = fmaf(-a, s[i], b * c[i]);
                        }
                    }
                }
                __syncwarp();
                const bool live = h + u < count && !padding;
                const float rs = normalizer<V>(v, n, inv_d, x);
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) {
                    x[i] *= rs;
                    if (live) dw[i] = fmaf(y[i], x[i], dw[i]); // eps = 0 makes the xhat of a row of zeros NaN
                    y[i] *= weights[i < V ? n.a + i : n.b + i - V];
                }
                if (v.norm != 0) {
                    const float sgx = group_sum(lane_dot(y, x), v.G) * inv_d;
                    const float sg = v.norm == 2 ? group_sum(lane_sum(y), v.G) * inv_d : 0.0f;
#pragma unroll
                    for (int i = 0; i < 2 * V; ++i) y[i] = rs * (fmaf(-x[i], sgx, y[i]) - sg);
                }
                if (h + u < count) {
                    if (padding) {
#pragma unroll
                        for (int i = 0; i < 2 * V; ++i) y[i] = 0.0f;
                    }
                    T* dst = reinterpret_cast<T*>(m.dx + static_cast<uint64_t>(static_cast<uint32_t>(u)) * sd.dx.h);
                    if (n.has_a) *reinterpret_cast<Raw*>(dst + n.a) = pack<T, VB>(y);
                    if (n.has_b) *reinterpret_cast<Raw*>(dst + n.b) = pack<T, VB>(y + V);
                }
            }
            m.dx += static_cast<uint64_t>(U) * sd.dx.h;
        }
    }
    if (!v.partial) return;
    // the rows of a warp, then the warps of the block in order: one line of the workspace per block
#pragma unroll
    for (int i = 0; i < 2 * V; ++i)
        for (int o = v.G; o < 32; o <<= 1) dw[i] += __shfl_xor_sync(0xffffffffu, dw[i], o);
    float* mine = sums + (threadIdx.x >> 5) * v.d;
    if (lane < v.G) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (n.has_a) mine[n.a + i] = dw[i];
            if (n.has_b) mine[n.b + i] = dw[V + i];
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < v.d; e += 256) {
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) t += sums[k * v.d + e];
        v.partial[static_cast<long long>(blockIdx.x) * v.d + e] = t;
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

void divisor(uint32_t d, uint32_t* mul, int* shift) {
    *mul = 0; *shift = 0;
    if (d <= 1) return;
    while (*shift < 30 && (2u << *shift) < d) ++*shift;
    *mul = static_cast<uint32_t>(((1ull << (32 + *shift)) + d - 1) / d);
}

template <typename T, int VB>
cudaError_t launch_vec(const QkParams& p, QkVec& v, bool backward, cudaStream_t st) {
    constexpr int V = VB / sizeof(T);
    const int chunks = p.d / V, half = p.interleaved ? 0 : p.rot / 2 / V;
    const int pairs = half + (chunks - 2 * half + 1) / 2;
    v.G = 1;
    while (v.G < pairs) v.G *= 2;
    v.all_turn = p.rot == p.d;
    v.table_vec = (reinterpret_cast<uintptr_t>(p.cos_t) | reinterpret_cast<uintptr_t>(p.sin_t)) % 16 == 0 && (p.rot / 2) % 4 == 0 &&
                  (!p.interleaved || (p.rot / 2) % V == 0);
    const int W = 32 / v.G, sms = num_sms();
    const long long tokens = static_cast<long long>(p.B) * p.L;
    // an item per token where that gives every SM 64 warps or more of them (a few rounds of what is resident), else the heads in
    // several items, of as many heads as are loaded at once
    const long long wanted = 64ll * sms * W;
    long long warps[2];
    for (int k = 0; k < 2; ++k) {
        QkSide& sd = v.side[k];
        const int H = k ? p.hk : p.hq;
        const long long cuts = std::min<long long>(std::max(H, 1), std::max(1ll, wanted / tokens));
        sd.H = H;
        sd.per_item = std::max(1, static_cast<int>((H + cuts - 1) / cuts));
        sd.per_item = std::min(std::max(H, 1), (sd.per_item + kHeadsAtOnce - 1) / kHeadsAtOnce * kHeadsAtOnce);
        sd.chunks = std::max(1, (H + sd.per_item - 1) / sd.per_item);
        sd.items = H ? static_cast<uint32_t>(tokens * sd.chunks) : 0u;
        divisor(static_cast<uint32_t>(sd.chunks), &sd.chunks_mul, &sd.chunks_shift);
        warps[k] = (static_cast<long long>(sd.items) + W - 1) / W;
    }
    // forward: blocks to fill the SMs eight times over; backward: few, as each leaves a line of weight gradients to be summed
    const long long cap = (backward ? 2ll : 8ll) * sms;
    long long bq = (warps[0] + 7) / 8, bk = (warps[1] + 7) / 8;
    if (bq + bk > cap) {                           // in proportion to the rows
        const long long share = cap * p.hq / (p.hq + p.hk);
        bq = bq ? std::min(bq, std::max(1ll, share)) : 0;
        bk = bk ? std::min(bk, std::max(1ll, cap - bq)) : 0;
    }
    v.side[0].blocks = static_cast<uint32_t>(bq); v.side[1].blocks = static_cast<uint32_t>(bk);
    const dim3 grid(static_cast<unsigned>(bq + bk));
    if (!backward) return launch_pdl(qk_vec_forward_kernel<T, VB, kHeadsAtOnce, V == 8 ? 2 : V == 4 ? 3 : 4>, grid, dim3(256), 0, st, v);
    cudaError_t e = launch_pdl(qk_vec_backward_kernel<T, VB, V == 8 ? 2 : 4, 2>, grid, dim3(256), v.partial ? 8u * p.d * sizeof(float) : 0u, st, v);
    if (e == cudaSuccess && v.partial)
        e = launch_pdl(qk_weight_sum_kernel, dim3((p.d + 31) / 32, 2), dim3(1024), 0, st, static_cast<const float*>(v.partial), static_cast<int>(bq),
                       static_cast<int>(bk), p.d, p.dqw, p.dkw);
    return e;
}

// The widest chunk that every base, stride and boundary of the call allows: 16, 8 or 4 bytes; 0 for none, or for strides beyond 32 bits.
int chunk_bytes(const QkParams& p, bool backward, int elem) {
    uint64_t bits = static_cast<uint64_t>(p.d) * elem, most = 0;
    if (p.rot > 0 && !p.interleaved) bits |= static_cast<uint64_t>(p.rot / 2) * elem;
    auto stride = [&](long long s, int extent) {
        if (extent <= 1) return;
        most = std::max(most, static_cast<uint64_t>(s));
        bits |= static_cast<uint64_t>(s) * elem;
    };
    auto add = [&](const HeadsView& h, int heads) {
        if (heads == 0) return;
        bits |= reinterpret_cast<uintptr_t>(h.p);
        stride(h.b, p.B); stride(h.l, p.L); stride(h.h, heads);
    };
    add(p.q, p.hq); add(p.k, p.hk); add(p.qo, p.hq); add(p.ko, p.hk);
    if (backward) { add(p.dq, p.hq); add(p.dk, p.hk); }
    if (most > UINT32_MAX / 4) return 0;
    for (int vb = 16; vb >= 4; vb /= 2)
        if (bits % vb == 0 && vb >= elem) return p.d * elem <= 64 * vb ? vb : 0;
    return 0;
}

template <typename T>
int launch_any(const QkParams& p, bool backward, cudaStream_t st) {
    const int vb = chunk_bytes(p, backward, sizeof(T));
    cudaError_t e;
    if (vb) {
        QkVec v{};
        auto view = [&](const HeadsView& h, int heads) {       // a stride of an extent of 1 is never used
            auto bytes = [](long long s, int n) { return n > 1 ? static_cast<uint32_t>(s * sizeof(T)) : 0u; };
            return QkView{static_cast<unsigned char*>(h.p), bytes(h.b, p.B), bytes(h.l, p.L), bytes(h.h, heads)};
        };
        for (int k = 0; k < 2; ++k) {
            const int H = k ? p.hk : p.hq;
            v.side[k].x = view(k ? p.k : p.q, H); v.side[k].y = view(k ? p.ko : p.qo, H); v.side[k].dx = view(k ? p.dk : p.dq, H);
            v.side[k].w = k ? p.kw : p.qw;
        }
        v.cos_t = p.cos_t; v.sin_t = p.sin_t; v.positions = p.positions; v.partial = p.partial; v.pos_b = p.pos_b;
        v.L = static_cast<uint32_t>(p.L); v.d = p.d; v.rot = p.rot; v.norm = p.norm; v.interleaved = p.interleaved; v.table_rows = p.table_rows;
        v.eps = p.eps;
        divisor(v.L, &v.l_mul, &v.l_shift);
        e = vb == 16 ? launch_vec<T, 16>(p, v, backward, st) : vb == 8 ? launch_vec<T, 8>(p, v, backward, st) : launch_vec<T, 4>(p, v, backward, st);
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
