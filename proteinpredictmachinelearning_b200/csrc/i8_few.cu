// i8_few.cu -- a Linear in 8-bit integers for a few tokens (a serving step): quantizer and product in one kernel.
//
// The weights are the traffic (N K bytes, each read once); a token's row is small, so every block quantizes all tokens for itself
// into shared memory while its first weights are on their way, instead of a kernel of its own doing it first.  A warp
// takes R output channels and sums them with dp4a against all tokens: 4 multiply-adds an instruction cover up to kI8Few tokens at
// the memory's rate.  16 bytes of a weight row per lane and step, kDeep steps of them on the way before the tokens are quantized;
// the integers of the tokens come from shared memory.  Each sum ends in a lane of its own, so that the scales are fetched and the
// results finished all at once (one after the other, 4 x 512 -> 8192 took 6.5 us for 3.8).
// Latency-bound: 1 x 1024 -> 4096 bf16 2.5 us from launch to launch, against 5.4 of the two kernels it replaces; 1 x 4096 -> 8192
// 9.0 us, 3.7 TB/s of weights.
#include "i8_common.cuh"

namespace ppml_b200 {
namespace {

constexpr int kFewThreads = 256, kFewWarps = 8;

__device__ __forceinline__ uint4 load16(const int8_t* row, int k, int k_vec) {
    return k < k_vec ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0, 0, 0, 0);
}
__device__ __forceinline__ int dot16(const uint4& a, const uint4& b, int acc) {
    acc = __dp4a(static_cast<int>(a.x), static_cast<int>(b.x), acc);
    acc = __dp4a(static_cast<int>(a.y), static_cast<int>(b.y), acc);
    acc = __dp4a(static_cast<int>(a.z), static_cast<int>(b.z), acc);
    return __dp4a(static_cast<int>(a.w), static_cast<int>(b.w), acc);
}

template <typename TX, typename TC, int MT, int R>
__global__ void __launch_bounds__(kFewThreads) i8_few_kernel(const TX* __restrict__ x, long long ld_x, const I8Product p) {
    constexpr int N = Vec16<TX>::kN, kPer = kFewThreads / MT, kWarpsPer = kPer / 32, kDeep = R == 1 ? 4 : 2;
    extern __shared__ __align__(16) int8_t xq[];   // [MT][K16]
    __shared__ uint32_t part[kFewWarps];
    __shared__ float scales[MT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int k16 = (p.K + 15) & ~15;
    const long long n0 = (static_cast<long long>(blockIdx.x) * kFewWarps + warp) * R;
    const int kw_vec = ((reinterpret_cast<uintptr_t>(p.B) | static_cast<uintptr_t>(p.ldb)) & 15) == 0 ? p.K & ~15 : 0;
    const int8_t* rows[R];
#pragma unroll
    for (int r = 0; r < R; ++r) rows[r] = p.B + min(n0 + r, static_cast<long long>(p.N) - 1) * p.ldb;
    pdl_wait();
    pdl_launch_dependents();
    uint4 w[kDeep][R];
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
#pragma unroll
        for (int r = 0; r < R; ++r) w[d][r] = load16(rows[r], 16 * lane + 512 * d, kw_vec);

    // lane r MT + m writes the value of channel r and token m
    const int my_m = lane % MT;
    const long long my_n = n0 + lane / MT;
    const bool owns = lane < R * MT && my_m < p.M && my_n < p.N;
    const float my_scale = owns ? p.b_scale[my_n] : 0.0f, my_bias = owns && p.bias ? p.bias[my_n] : 0.0f;

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
    for (int k0 = 16 * lane; k0 < kw_vec; k0 += 512 * kDeep) {
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            const int k = k0 + 512 * d;
            if (k < kw_vec) {
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const uint4 a = *reinterpret_cast<const uint4*>(xq + m * k16 + k);
#pragma unroll
                    for (int r = 0; r < R; ++r) acc[r][m] = dot16(a, w[d][r], acc[r][m]);
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r) w[d][r] = load16(rows[r], k + 512 * kDeep, kw_vec);
        }
    }
    for (int k = kw_vec + lane; k < p.K; k += 32) {        // the last K % 16 values; all of them for unaligned weights
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[r][m] += rows[r][k] * xq[m * k16 + k];
    }
    int mine = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int sum = __reduce_add_sync(0xffffffffu, acc[r][m]);
            mine = lane == r * MT + m ? sum : mine;
        }
    if (owns) {
        float y = i8_epilogue(mine, scales[my_m], my_scale, my_bias, p);
        if (p.gate) y *= to_f32(static_cast<const TC*>(p.gate)[my_m * p.ld_gate + my_n]);
        static_cast<TC*>(p.C)[my_m * p.ldc + my_n] = from_f32<TC>(y);
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
    // Two channels a warp: half the blocks quantize the tokens again, with 2 x 1 KB on the way for each warp; one channel a warp (four
    // steps of it on the way) where the rows are long and the blocks are two an SM at most.  One and two channels measured: 1 x 1024 ->
    // 1024 2.5 and 2.2 us, 1 x 1024 -> 8192 5.3 and 3.5, 4 x 2048 -> 8192 10.4 and 8.0; 1 x 4096 -> 2048 4.6 and 5.7, 4 x 2048 -> 1024
    // 3.6 and 3.9.  Four channels gained 0.2 us at 4 x 1024 -> 4096 and lost as much elsewhere.
    return p.K > 1024 && p.N <= 2 * kFewWarps * num_sms() ? launch_r<TX, TC, MT, 1>(x, ld_x, p, st) : launch_r<TX, TC, MT, 2>(x, ld_x, p, st);
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

// Up to four tokens, as long as quantizing them in every block costs less than a kernel before the product (us this way and in two
// kernels): 4 x 2048 -> 1024 3.6 and 5.7, 4 x 2048 -> 8192 8.0 and 8.3, 2 x 4096 -> 8192 9.6 and 11.0; with 16384 values 4 x 4096 -> 4096
// 9.6 and 8.4, 1 x 16384 -> 1024 11.9 and 10.4.
bool i8_few(long long M, int K) { return M <= kI8Few && (M <= 2 ? M : 4) * ((K + 15ll) / 16 * 16) <= kI8FewValues; }

int launch_i8_few(const void* x, int x_type, long long ld_x, const I8Product& p, cudaStream_t st) {
    switch (x_type) {
        case kTypeF32: return launch_c(static_cast<const float*>(x), ld_x, p, st);
        case kTypeF16: return launch_c(static_cast<const __half*>(x), ld_x, p, st);
        default: return launch_c(static_cast<const __nv_bfloat16*>(x), ld_x, p, st);
    }
}

}  // namespace ppml_b200
