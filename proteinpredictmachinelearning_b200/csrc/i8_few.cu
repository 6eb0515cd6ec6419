// i8_few.cu -- a Linear in 8-bit integers for a few tokens (a serving step): quantizer and product in one kernel.
//
// The weights are the traffic (N K bytes, each read once); a token's row is small, so every block quantizes all tokens for itself
// into shared memory while its first weights are on their way, instead of a kernel of its own doing it first.  A warp
// takes R output channels and sums them with dp4a against all tokens: 4 multiply-adds an instruction cover up to kI8Few tokens at
// the memory's rate.  16 bytes of a weight row per lane and step; the integers of the tokens come from shared memory.
// Latency-bound: 1 x 1024 -> 4096 bf16 3.2 us from launch to launch, against 6.3 of the two kernels it replaces.
#include "i8_common.cuh"

namespace ppml_b200 {
namespace {

constexpr int kFewThreads = 256, kFewWarps = 8;

__device__ __forceinline__ uint4 load16(const int8_t* row, int k, int K, bool vec) {
    if (vec && k + 16 <= K) return *reinterpret_cast<const uint4*>(row + k);
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i)
        if (k + i < K) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i & 3));
    return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int acc) {
    acc = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), acc);
    acc = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), acc);
    acc = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), acc);
    return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), acc);
}

template <typename TX, typename TC, int MT, int R>
__global__ void __launch_bounds__(kFewThreads) i8_few_kernel(const TX* __restrict__ x, long long ld_x, const I8Product p) {
    constexpr int N = Vec16<TX>::kN, kPer = kFewThreads / MT, kWarpsPer = kPer / 32;
    extern __shared__ __align__(16) int8_t xq[];   // [MT][K16]
    __shared__ uint32_t part[kFewWarps];
    __shared__ float scales[MT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int k16 = (p.K + 15) & ~15;
    const long long n0 = (static_cast<long long>(blockIdx.x) * kFewWarps + warp) * R;
    const bool w_vec = ((reinterpret_cast<uintptr_t>(p.B) | static_cast<uintptr_t>(p.ldb)) & 15) == 0;
    const int8_t* rows[R];
#pragma unroll
    for (int r = 0; r < R; ++r) rows[r] = p.B + min(n0 + r, static_cast<long long>(p.N) - 1) * p.ldb;
    pdl_wait();
    pdl_launch_dependents();
    uint4 w[R];
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = load16(rows[r], 16 * lane, p.K, w_vec);

    // kPer threads on each token
    {
        const int m = threadIdx.x / kPer, me = threadIdx.x % kPer;
        const TX* xr = x + (m < p.M ? m : 0) * ld_x;
        const bool x_vec = ((reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(ld_x * sizeof(TX))) & 15) == 0;
        const int k_vec = x_vec ? p.K / N * N : 0;
        uint32_t top = 0;
        for (int k = me * N; k < k_vec; k += kPer * N) top = max(top, top_of<TX>(*reinterpret_cast<const uint4*>(xr + k)));
        for (int k = k_vec + me; k < p.K; k += kPer) top = max(top, magnitude_bits(to_f32(xr[k])));
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) part[warp] = top;
        __syncthreads();
        top = 0;
#pragma unroll
        for (int i = 0; i < kWarpsPer; ++i) top = max(top, part[m * kWarpsPer + i]);
        const float s = i8_scale(top), inv = i8_inverse(s);
        int8_t* q = xq + m * k16;
        for (int k = me * N; k < k_vec; k += kPer * N) {
            uint32_t b[N / 4];
            quantize_vec<TX>(*reinterpret_cast<const uint4*>(xr + k), s, inv, b);
#pragma unroll
            for (int i = 0; i < N / 4; ++i) reinterpret_cast<uint32_t*>(q + k)[i] = b[i];
        }
        for (int k = k_vec + me; k < k16; k += kPer) q[k] = k < p.K ? static_cast<int8_t>(i8_quantize(to_f32(xr[k]), s)) : 0;
        if (me == 0) scales[m] = s;
        __syncthreads();
    }

    int acc[R][MT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[r][m] = 0;
    for (int k = 16 * lane; k < p.K; k += 512) {
        uint4 next[R];
#pragma unroll
        for (int r = 0; r < R; ++r) next[r] = k + 512 < p.K ? load16(rows[r], k + 512, p.K, w_vec) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const uint4 a = *reinterpret_cast<const uint4*>(xq + m * k16 + k);
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][m] = dot16(a, w[r], acc[r][m]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) w[r] = next[r];
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int sum = __reduce_add_sync(0xffffffffu, acc[r][m]);
            const long long n = n0 + r;
            if (lane == r * MT + m && n < p.N && m < p.M) {
                float y = i8_epilogue(sum, scales[m], p.b_scale[n], p.bias ? p.bias[n] : 0.0f, p.act);
                if (p.gate) y *= to_f32(static_cast<const TC*>(p.gate)[m * p.ld_gate + n]);
                static_cast<TC*>(p.C)[m * p.ldc + n] = from_f32<TC>(y);
            }
        }
}

template <typename TX, typename TC, int MT, int R>
cudaError_t launch_r(const TX* x, long long ld_x, const I8Product& p, cudaStream_t st) {
    const long long per = kFewWarps * R;
    return launch_pdl(i8_few_kernel<TX, TC, MT, R>, dim3(static_cast<unsigned>((p.N + per - 1) / per)), dim3(kFewThreads),
                      static_cast<size_t>(MT) * ((p.K + 15) / 16 * 16), st, x, ld_x, p);
}
template <typename TX, typename TC, int MT>
cudaError_t launch_m(const TX* x, long long ld_x, const I8Product& p, cudaStream_t st) {
    // About two blocks an SM: every block quantizes the tokens again, and every warp should have its weights on the way at once.
    // Measured with 1 and with 4 channels a warp: 1 x 1024 -> 1024 2.5 and 3.2 us, 3 x 2048 -> 2048 4.6 and 6.7, 1 x 4096 -> 8192
    // 14.6 and 10.4.
    const long long blocks = 2ll * num_sms();
    if (p.N <= kFewWarps * blocks) return launch_r<TX, TC, MT, 1>(x, ld_x, p, st);
    if (p.N <= 2 * kFewWarps * blocks) return launch_r<TX, TC, MT, 2>(x, ld_x, p, st);
    return launch_r<TX, TC, MT, 4>(x, ld_x, p, st);
}
template <typename TX, typename TC>
int launch_x(const TX* x, long long ld_x, const I8Product& p, cudaStream_t st) {
    const cudaError_t e = p.M == 1 ? launch_m<TX, TC, 1>(x, ld_x, p, st) : p.M == 2 ? launch_m<TX, TC, 2>(x, ld_x, p, st) : launch_m<TX, TC, 4>(x, ld_x, p, st);
    if (e != cudaSuccess) { cudaGetLastError(); return ST_LAUNCH; }
    return ST_OK;
}
template <typename TX>
int launch_c(const TX* x, long long ld_x, const I8Product& p, cudaStream_t st) {
    return p.c_type == kTypeF32 ? launch_x<TX, float>(x, ld_x, p, st)
                                : p.c_type == kTypeF16 ? launch_x<TX, __half>(x, ld_x, p, st) : launch_x<TX, __nv_bfloat16>(x, ld_x, p, st);
}

}  // namespace

// Up to four tokens, as long as quantizing them in every block costs less than a kernel before the product: 2 x 4096 -> 8192 takes
// 11.5 us this way and 11.2 in two kernels, 1 x 4096 -> 8192 10.4 and 11.1, 4 x 8192 -> 1024 15 and 8.
bool i8_few(long long M, int K) { return M <= kI8Few && (M <= 2 ? M : 4) * ((K + 15ll) / 16 * 16) <= kI8FewValues; }

int launch_i8_few(const void* x, int x_type, long long ld_x, const I8Product& p, cudaStream_t st) {
    switch (x_type) {
        case kTypeF32: return launch_c(static_cast<const float*>(x), ld_x, p, st);
        case kTypeF16: return launch_c(static_cast<const __half*>(x), ld_x, p, st);
        default: return launch_c(static_cast<const __nv_bfloat16*>(x), ld_x, p, st);
    }
}

}  // namespace ppml_b200
