// qk_norm_rope.cu -- norms of queries and keys for each head with the position rotation in the same pass, and the backward pass.
//
//   xhat = (x - mu) * r,  r = 1 / sqrt(mean((x - mu)^2) + eps)     over one head of one token (mu = 0 for the root mean square)
//   n    = xhat * w
//   y    = n with its first `rot` dims rotated: (a, b) -> (a cos - b sin, b cos + a sin), pairs (i, i + rot / 2) or (2 i, 2 i + 1)
// Backward, from x and dy alone (nothing is kept by the forward pass):
//   g    = dy with the rotation turned back,  dw = sum over tokens and heads of g * xhat,  gh = g * w
//   dx   = r * (gh - mean(gh) - xhat * mean(gh * xhat))            (without the mean(gh) term for the root mean square)
// All of it in fp32, rounded once where a result is stored.  The bytes of Q, K and their results are what a pass cannot do without; with
// 16-byte chunks and a power of two of lanes a row it is bound by them (5.2 - 6.2 TB/s forward), elsewhere by the pieces it reads them in:
// 2^26 values in bf16, forward, TB/s: head dim 8 1.7, 16 3.4, 32 5.2, 40 3.1, 48 and 96 4.7, 64 - 512 5.5 - 5.7, 80 4.3, 46 0.5, 126 1.1.
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
    int d, rot, norm, interleaved, table_rows, table_vec;
    int all_turn, full;                            // every value turns; every lane holds 2 V values
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
// exchange between lanes, and two values go by one packed instruction.  G lanes (a power of two) hold a row, a warp 32 / G of
// them, of different tokens: each group of lanes walks over the heads of its token, so that the position, its table row and
// all but one addition of an address are had once per token instead of once per row.  A block works on one side (Q or K).
// What bounds it: the bytes in flight.  Rows wait in registers from the load to the store, and 16 (bf16) to 24 (fp32) warps an SM are
// what that leaves; a ring of rows in shared memory (cp.async) kept more in flight and cost 40 instructions a row: at an earlier
// step 120 against 122 us on the long case below, 43 against 34 on the short one, and was dropped.
// Measured (forward): 65536 tokens x 16 heads of 32, fp32 44 us (6.1 TB/s); 32768 tokens x 40 heads of 128, bf16 115 us (5.9 TB/s);
// 16384 tokens x 32 heads of 64, bf16, LayerNorm, neighbouring pairs 30 us; backward of the last 47 us (4.3 TB/s), of 16384 tokens x 16
// heads of 32, fp32 23 us.
constexpr int kHeadsAtOnce = 4;                    // rows of a group of lanes that are loaded together (forward)

template <int VB> struct RawOf;
template <> struct RawOf<16> { using type = uint4; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<4> { using type = uint32_t; };

// The lane's 2 V values as V packed pairs: pair j holds values 2 j and 2 j + 1 of its two chunks one behind the other (V = 1: one of
// each).  All arithmetic goes by packed instructions.
template <typename T> __device__ __forceinline__ uint64_t widen(uint32_t two) {
    if constexpr (sizeof(T) == 2) {
        const uint16_t lo = static_cast<uint16_t>(two & 0xffffu), hi = static_cast<uint16_t>(two >> 16);
        return pack2(to_f32(*reinterpret_cast<const T*>(&lo)), to_f32(*reinterpret_cast<const T*>(&hi)));
    }
    return 0;
}
// n / d for n < 2^31: with 2^s < d <= 2^(s + 1) and m = ceil(2^(32 + s) / d) the error m d - 2^(32 + s) is below 2^(s + 1), so that
// (n m) >> (32 + s) is exact; d = 1 has m = 0.
__device__ __forceinline__ uint32_t div_by(uint32_t n, uint32_t m, int s) { return m == 0 ? n : __umulhi(n, m) >> s; }

// 1 / sqrt(v): the hardware's estimate (2 units in the last place) and one Newton step, which leaves its rounding errors alone; a
// division and a square root take 40 instructions.  0 and infinity stay what the estimate makes of them.
__device__ __forceinline__ float inv_sqrt(float v) {
    const float r = rsqrtf(v);
    return r > 0.0f && r < __uint_as_float(0x7f800000u) ? fmaf(0.5f * r, fmaf(-v * r, r, 1.0f), r) : r;
}

// This lane's part of a row (element and byte offsets of its chunks) and where its pairs stand in the table.
struct Lane { int a, b, pair, turning; uint32_t at_a, at_b; bool has_a, has_b; };      // turning: packed pairs that turn
template <typename T, int VB> __device__ __forceinline__ Lane lane_of(const QkVec& v, int l) {
    constexpr int V = VB / sizeof(T);
    Lane n;
    const int chunks = v.d / V, half = v.interleaved ? 0 : v.rot / 2 / V;
    const bool halves = l < half;
    const int a = halves ? l : 2 * half + 2 * (l - half), b = halves ? l + half : a + 1;
    n.has_a = a < chunks; n.has_b = b < chunks;
    n.pair = l * V;
    n.turning = v.interleaved ? min(max(v.rot / 2 - n.pair, 0), V) : halves ? V : 0;
    n.a = a * V; n.b = b * V;
    n.at_a = static_cast<uint32_t>(a * VB); n.at_b = static_cast<uint32_t>(b * VB);
    return n;
}
// cos and sin of the lane's pairs; NaN beyond the table; 1 and 0 where nothing turns and, without a look-up, at a negative position
// (padding, and lanes without an item): a row that no token names may hold anything, and 0 times a NaN would reach the weight gradients
template <int V> __device__ __forceinline__ void load_table(const QkVec& v, const Lane& n, int pos, float (&c)[V], float (&s)[V]) {
    const int half = v.rot / 2;
    const float none = pos >= v.table_rows ? __uint_as_float(0x7fffffffu) : 1.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) { c[i] = i < n.turning ? none : 1.0f; s[i] = 0.0f; }
    if (n.turning == 0 || pos < 0 || pos >= v.table_rows) return;
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
            if (i < n.turning) { c[i] = v.cos_t[at + i]; s[i] = v.sin_t[at + i]; }     // neighbours: may end inside the chunk
    }
}
// Sum over the lanes of a row; LG >= 0: their number is 2^LG, else G (a branch per step).
template <int LG> __device__ __forceinline__ float group_sum(float v, int G) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
        if (LG >= 0 ? o < (1 << (LG >= 0 ? LG : 0)) : o < G) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int N> __device__ __forceinline__ float lane_sum(const uint64_t (&x)[N]) {
    uint64_t t = x[0];
#pragma unroll
    for (int j = 1; j < N; ++j) t = fadd2(t, x[j]);
    float a, b; unpack2(t, a, b);
    return a + b;
}
template <int N> __device__ __forceinline__ float lane_dot(const uint64_t (&x)[N], const uint64_t (&y)[N]) {
    uint64_t t = fmul2(x[0], y[0]);
#pragma unroll
    for (int j = 1; j < N; ++j) t = ffma2(x[j], y[j], t);
    float a, b; unpack2(t, a, b);
    return a + b;
}
// x becomes x - mean; returns 1 / sqrt(..) of the row.  Values that do not exist stay 0.
template <int V, int LG> __device__ __forceinline__ float normalizer(const QkVec& v, const Lane& n, float inv_d, uint64_t (&x)[V]) {
    if (v.norm == 0) return 1.0f;
    if (v.norm == 2) {
        const float m = group_sum<LG>(lane_sum(x), v.G) * inv_d;
        const uint64_t m2 = pack2(-m, -m);
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = fadd2(x[j], m2);
        if (!v.full) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float lo, hi; unpack2(x[j], lo, hi);
                x[j] = pack2((V == 1 || 2 * j < V ? n.has_a : n.has_b) ? lo : 0.0f, (2 * j + 1 < V ? n.has_a : n.has_b) ? hi : 0.0f);
            }
        }
    }
    return inv_sqrt(fmaf(group_sum<LG>(lane_dot(x, x), v.G), inv_d, v.eps));
}
__device__ __forceinline__ uint64_t swap2(uint64_t p) { float a, b; unpack2(p, a, b); return pack2(b, a); }
// y = x * c + partner * s.  The partner of a packed pair is the same place of the other chunk, or with neighbouring pairs (and with
// V = 1) its own two values exchanged.  Pairs that do not turn are only scaled: an infinity must not meet a neighbour, not even
// times 0.
template <int V> __device__ __forceinline__ void turn(const QkVec& v, const Lane& n, const uint64_t (&x)[V], const uint64_t (&c)[V], const uint64_t (&s)[V],
                                                      uint64_t (&y)[V]) {
#pragma unroll
    for (int j = 0; j < V; ++j) y[j] = fmul2(x[j], c[j]);
    if (v.all_turn) {
        if (V == 1 || v.interleaved) {
#pragma unroll
            for (int j = 0; j < V; ++j) y[j] = ffma2(swap2(x[j]), s[j], y[j]);
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) y[j] = ffma2(x[(j + V / 2) % V], s[j], y[j]);
        }
    } else if (V == 1 || v.interleaved) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n.turning) y[j] = ffma2(swap2(x[j]), s[j], y[j]);
    } else if (n.turning) {
#pragma unroll
        for (int j = 0; j < V; ++j) y[j] = ffma2(x[(j + V / 2) % V], s[j], y[j]);
    }
}
// The factors of turn() from the lane's cos and sin and the weights of its values.
template <int V> __device__ __forceinline__ void factors(const QkVec& v, const Lane& n, int pos, const float* weights, uint64_t (&c)[V], uint64_t (&s)[V]) {
    float cs[V], sn[V];
    load_table<V>(v, n, pos, cs, sn);
    if (V == 1 || v.interleaved) {                 // the lane's values are one run of V pairs (V = 1: one value of each chunk)
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float w0 = weights[n.a + 2 * j], w1 = V == 1 ? weights[n.b] : weights[n.a + 2 * j + 1];
            c[j] = pack2(w0 * cs[j], w1 * cs[j]);
            s[j] = pack2(-w1 * sn[j], w0 * sn[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const float c0 = cs[2 * j], c1 = cs[2 * j + 1], s0 = sn[2 * j], s1 = sn[2 * j + 1];
            const float a0 = weights[n.a + 2 * j], a1 = weights[n.a + 2 * j + 1], b0 = weights[n.b + 2 * j], b1 = weights[n.b + 2 * j + 1];
            c[j] = pack2(a0 * c0, a1 * c1); c[V / 2 + j] = pack2(b0 * c0, b1 * c1);
            s[j] = pack2(-b0 * s0, -b1 * s1); s[V / 2 + j] = pack2(a0 * s0, a1 * s1);
        }
    }
}
// Turns a gradient back, in place, from the lane's cos and sin alone (half the registers of factors()).
template <int V> __device__ __forceinline__ void turn_back(const QkVec& v, const Lane& n, const float (&c)[V], const float (&s)[V], uint64_t (&y)[V]) {
    auto neighbours = [&](int j) {
        float a, b;
        unpack2(y[j], a, b);
        y[j] = pack2(fmaf(b, s[j], a * c[j]), fmaf(-a, s[j], b * c[j]));
    };
    auto halves = [&]() {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const uint64_t c2 = pack2(c[2 * j], c[2 * j + 1]), s2 = pack2(s[2 * j], s[2 * j + 1]), a = y[j], b = y[V / 2 + j];
            const uint64_t minus = pack2(-s[2 * j], -s[2 * j + 1]);
            y[j] = ffma2(b, s2, fmul2(a, c2));
            y[V / 2 + j] = ffma2(a, minus, fmul2(b, c2));
        }
    };
    if (v.all_turn) {
        if (V == 1 || v.interleaved) {
#pragma unroll
            for (int j = 0; j < V; ++j) neighbours(j);
        } else {
            halves();
        }
    } else if (V == 1 || v.interleaved) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < n.turning) neighbours(j);
    } else if (n.turning) {
        halves();
    }
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

// the two chunks of a row as packed pairs
template <typename T, int VB> __device__ __forceinline__ void pairs_of(const typename RawOf<VB>::type& a, const typename RawOf<VB>::type& b,
                                                                       uint64_t (&x)[VB / sizeof(T)]) {
    constexpr int V = VB / sizeof(T), kWords = VB / 4;
    uint32_t w[2 * kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) { w[i] = reinterpret_cast<const uint32_t*>(&a)[i]; w[kWords + i] = reinterpret_cast<const uint32_t*>(&b)[i]; }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if constexpr (sizeof(T) == 2) x[j] = widen<T>(w[j]);
        else x[j] = pack2(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
    }
}
// Predicated accesses: a row's two dozen conditions would be branches otherwise.
template <int VB> __device__ __forceinline__ typename RawOf<VB>::type load_raw(const unsigned char* p, bool yes) {
    typename RawOf<VB>::type r;
    const int on = yes;
    if constexpr (VB == 16)
        asm volatile("{.reg .pred p; setp.ne.s32 p, %5, 0; mov.b32 %0, 0; mov.b32 %1, 0; mov.b32 %2, 0; mov.b32 %3, 0; "
                     "@p ld.global.v4.b32 {%0, %1, %2, %3}, [%4];}" : "=&r"(r.x), "=&r"(r.y), "=&r"(r.z), "=&r"(r.w) : "l"(p), "r"(on) : "memory");
    else if constexpr (VB == 8)
        asm volatile("{.reg .pred p; setp.ne.s32 p, %3, 0; mov.b32 %0, 0; mov.b32 %1, 0; @p ld.global.v2.b32 {%0, %1}, [%2];}"
                     : "=&r"(r.x), "=&r"(r.y) : "l"(p), "r"(on) : "memory");
    else asm volatile("{.reg .pred p; setp.ne.s32 p, %2, 0; mov.b32 %0, 0; @p ld.global.b32 %0, [%1];}" : "=&r"(r) : "l"(p), "r"(on) : "memory");
    return r;
}
template <int VB> __device__ __forceinline__ void store_raw(unsigned char* p, const typename RawOf<VB>::type& r, bool yes) {
    const int on = yes;
    if constexpr (VB == 16)
        asm volatile("{.reg .pred p; setp.ne.s32 p, %5, 0; @p st.global.v4.b32 [%4], {%0, %1, %2, %3};}" ::"r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w), "l"(p), "r"(on) : "memory");
    else if constexpr (VB == 8)
        asm volatile("{.reg .pred p; setp.ne.s32 p, %3, 0; @p st.global.v2.b32 [%2], {%0, %1};}" ::"r"(r.x), "r"(r.y), "l"(p), "r"(on) : "memory");
    else asm volatile("{.reg .pred p; setp.ne.s32 p, %2, 0; @p st.global.b32 [%1], %0;}" ::"r"(r), "l"(p), "r"(on) : "memory");
}
template <typename T, int VB> __device__ __forceinline__ void store_pairs(const uint64_t (&y)[VB / sizeof(T)], unsigned char* to, uint32_t a, uint32_t b, bool has_a, bool has_b) {
    constexpr int V = VB / sizeof(T), kWords = VB / 4;
    uint32_t w[2 * kWords];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float lo, hi;
        unpack2(y[j], lo, hi);
        if constexpr (sizeof(T) == 2) w[j] = narrow2(lo, hi, T());
        else { w[2 * j] = __float_as_uint(lo); w[2 * j + 1] = __float_as_uint(hi); }
    }
    typename RawOf<VB>::type ra, rb;
#pragma unroll
    for (int i = 0; i < kWords; ++i) { reinterpret_cast<uint32_t*>(&ra)[i] = w[i]; reinterpret_cast<uint32_t*>(&rb)[i] = w[kWords + i]; }
    store_raw<VB>(to + a, ra, has_a);
    store_raw<VB>(to + b, rb, has_b);
}

// U rows of every group of lanes are requested together.
template <typename T, int VB, int U, int BLOCKS, int LG>
__global__ void __launch_bounds__(256, BLOCKS) qk_vec_forward_kernel(const __grid_constant__ QkVec v) {
    constexpr int V = VB / sizeof(T);
    using Raw = typename RawOf<VB>::type;
    __shared__ __align__(16) float weights[kQkMaxDim + 32];  // a lane past the end of a row reads behind it
    pdl_wait();
    pdl_launch_dependents();
    const bool key = blockIdx.x >= v.side[0].blocks;
    const QkSide& sd = v.side[key];
    const int lane = threadIdx.x & 31, W = 32 / v.G;
    const Lane n = lane_of<T, VB>(v, lane & (v.G - 1));
    const float inv_d = 1.0f / static_cast<float>(v.d);
    const uint32_t warp = (blockIdx.x - (key ? v.side[0].blocks : 0u)) * 8u + (threadIdx.x >> 5), step = sd.blocks * 8u * W;
    for (int e = threadIdx.x; e < kQkMaxDim + 32; e += 256) weights[e] = sd.w && e < v.d ? sd.w[e] : 1.0f;
    __syncthreads();
    for (uint32_t first = warp * W; first < sd.items; first += step) {
        Item m = item_of<false>(v, sd, first + lane / v.G);
        const int count = m.pos < 0 ? 0 : m.h1 - m.h0;         // padding is neither read nor written
        Raw ra[U], rb[U];
        auto load = [&](int h) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                ra[u] = load_raw<VB>(m.x + n.at_a, n.has_a && h + u < count);
                rb[u] = load_raw<VB>(m.x + n.at_b, n.has_b && h + u < count);
                m.x += sd.x.h;
            }
        };
        load(0);                                               // before the table, whose row waits for the position
        uint64_t c[V], s[V];
        factors<V>(v, n, m.pos, weights, c, s);
        for (int h = 0;;) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint64_t x[V], y[V];
                pairs_of<T, VB>(ra[u], rb[u], x);
                const float rs = normalizer<V, LG>(v, n, inv_d, x);
                const uint64_t r2 = pack2(rs, rs);
#pragma unroll
                for (int j = 0; j < V; ++j) x[j] = fmul2(x[j], r2);
                turn<V>(v, n, x, c, s, y);
                store_pairs<T, VB>(y, m.y, n.at_a, n.at_b, n.has_a && h + u < count, n.has_b && h + u < count);
                m.y += sd.y.h;
            }
            h += U;
            if (h >= sd.per_item) break;
            load(h);
        }
    }
}

template <typename T, int VB, int U, int BLOCKS, int LG>
__global__ void __launch_bounds__(256, BLOCKS) qk_vec_backward_kernel(const __grid_constant__ QkVec v) {
    constexpr int V = VB / sizeof(T);
    using Raw = typename RawOf<VB>::type;
    extern __shared__ float sums[];                // [8][d]
    __shared__ __align__(16) float weights[kQkMaxDim + 32];
    pdl_wait();
    pdl_launch_dependents();
    const bool key = blockIdx.x >= v.side[0].blocks;
    const QkSide& sd = v.side[key];
    const int lane = threadIdx.x & 31, W = 32 / v.G;
    const Lane n = lane_of<T, VB>(v, lane & (v.G - 1));
    const float inv_d = 1.0f / static_cast<float>(v.d);
    const uint32_t warp = (blockIdx.x - (key ? v.side[0].blocks : 0u)) * 8u + (threadIdx.x >> 5), step = sd.blocks * 8u * W;
    for (int e = threadIdx.x; e < kQkMaxDim + 32; e += 256) weights[e] = sd.w && e < v.d ? sd.w[e] : 1.0f;
    __syncthreads();
    uint64_t dw[V];
#pragma unroll
    for (int j = 0; j < V; ++j) dw[j] = pack2(0.0f, 0.0f);
    for (uint32_t first = warp * W; first < sd.items; first += step) {
        Item m = item_of<true>(v, sd, first + lane / v.G);
        const int count = m.h1 - m.h0, live = m.pos < 0 ? 0 : count;
        Raw ra[U], rb[U], ga[U], gb[U];
        auto load = [&](int h) {
#pragma unroll
            for (int u = 0; u < U; ++u) {          // padding may hold anything: its gradients are 0
                ra[u] = load_raw<VB>(m.x + n.at_a, n.has_a && h + u < live);
                rb[u] = load_raw<VB>(m.x + n.at_b, n.has_b && h + u < live);
                ga[u] = load_raw<VB>(m.y + n.at_a, n.has_a && h + u < live);
                gb[u] = load_raw<VB>(m.y + n.at_b, n.has_b && h + u < live);
                m.x += sd.x.h; m.y += sd.y.h;
            }
        };
        load(0);                                   // before the table, whose row waits for the position
        float c[V], s[V];
        load_table<V>(v, n, m.pos, c, s);
        for (int h = 0;;) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint64_t x[V], y[V];
                pairs_of<T, VB>(ra[u], rb[u], x);
                pairs_of<T, VB>(ga[u], gb[u], y);
                turn_back<V>(v, n, c, s, y);
                __syncwarp();
                float rs = normalizer<V, LG>(v, n, inv_d, x);
                if (h + u >= live) rs = 0.0f;      // a row of zeros then: with eps = 0 its xhat would be NaN
                const uint64_t r2 = pack2(rs, rs);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    x[j] = fmul2(x[j], r2);
                    dw[j] = ffma2(y[j], x[j], dw[j]);
                    const float w0 = V == 1 || 2 * j < V ? weights[n.a + 2 * j] : weights[n.b + 2 * j - V];
                    const float w1 = 2 * j + 1 < V ? weights[n.a + 2 * j + 1] : weights[n.b + 2 * j + 1 - V];
                    y[j] = fmul2(y[j], pack2(w0, w1));
                }
                if (v.norm != 0) {
                    const float sgx = -group_sum<LG>(lane_dot(y, x), v.G) * inv_d;
                    const float sg = v.norm == 2 ? -rs * group_sum<LG>(lane_sum(y), v.G) * inv_d : 0.0f;
                    const uint64_t sgx2 = pack2(sgx, sgx), sg2 = pack2(sg, sg);
#pragma unroll
                    for (int j = 0; j < V; ++j) y[j] = ffma2(ffma2(x[j], sgx2, y[j]), r2, sg2);
                }
                if (h + u >= live) {               // padding: 0 even under weights that are not finite
#pragma unroll
                    for (int j = 0; j < V; ++j) y[j] = 0;
                }
                store_pairs<T, VB>(y, m.dx, n.at_a, n.at_b, n.has_a && h + u < count, n.has_b && h + u < count);
                m.dx += sd.dx.h;
            }
            h += U;
            if (h >= sd.per_item) break;
            load(h);
        }
    }
    if (!v.partial) return;
    // the rows of a warp, then the warps of the block in order: one line of the workspace per block
    float* mine = sums + (threadIdx.x >> 5) * v.d;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float t[2];
        unpack2(dw[j], t[0], t[1]);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            for (int o = v.G; o < 32; o <<= 1) t[k] += __shfl_xor_sync(0xffffffffu, t[k], o);
            const bool in_a = 2 * j + k < V;
            if (lane < v.G && (in_a ? n.has_a : n.has_b)) mine[in_a ? n.a + 2 * j + k : n.b + 2 * j + k - V] = t[k];
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
    v.full = v.G * 2 * V == p.d;
    v.table_vec = (reinterpret_cast<uintptr_t>(p.cos_t) | reinterpret_cast<uintptr_t>(p.sin_t)) % 16 == 0 && (p.rot / 2) % 4 == 0 &&
                  (!p.interleaved || (p.rot / 2) % V == 0);
    const int W = 32 / v.G, sms = num_sms();
    const long long tokens = static_cast<long long>(p.B) * p.L;
    // An item is a token with all heads of a side, or, where tokens are few, with some of them.  What an item costs beside its rows
    // (position, table, factors: about two rows' work) speaks for long ones, even shares of the resident warps for many.
    // Measured on 16384 tokens x 16 heads of 64 (bf16): forward 30.0 us from 24 items' warps an SM, 31.1 from 48; backward,
    // whose grid is what is resident, 51.5 from 24 and 47.1 from 96.
    const long long wanted = (backward ? 96ll : 24ll) * sms * W;
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
    // rows at once and blocks an SM: as many as the registers hold without spilling; the lanes of a row are known to the instances
    // with 16-byte chunks
    constexpr int kForward = V == 8 ? 2 : V == 4 ? 3 : 4, kBackwardRows = V == 8 ? 2 : 4;
    const size_t lines = v.partial ? 8u * p.d * sizeof(float) : 0u;
    cudaError_t e;
#define PPML_LG(LG) e = backward ? launch_pdl(qk_vec_backward_kernel<T, VB, kBackwardRows, 2, LG>, grid, dim3(256), lines, st, v) \
                                 : launch_pdl(qk_vec_forward_kernel<T, VB, kHeadsAtOnce, kForward, LG>, grid, dim3(256), 0, st, v)
    if constexpr (VB == 16) {
        switch (v.G) {
            case 1: PPML_LG(0); break;
            case 2: PPML_LG(1); break;
            case 4: PPML_LG(2); break;
            case 8: PPML_LG(3); break;
            case 16: PPML_LG(4); break;
            default: PPML_LG(5);
        }
    } else {
        PPML_LG(-1);
    }
#undef PPML_LG
    if (!backward) return e;
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
