// i8_simt.cu -- 8-bit integers with a scale per token and per output channel on CUDA cores: the token quantizer, and the
// product for operands that TMA cannot address (a row pitch or a base off 16 bytes) and for PATH_SIMT.
#include "i8_common.cuh"

namespace ppml_b200 {
namespace {

// ---- quantizer: one pass over x ----
// A row's 16-byte pieces are all requested at once and stay in registers from the maximum to the quotients.  Bound by bandwidth
// (e + 1 bytes a value): 65536 x 256 fp32 13.8 us (6.1 TB/s).  Two forms:
// short rows: R rows per warp, no barrier; the two quotients of a row (20 instructions) are taken by R lanes at once.
template <typename T, int NV, int R>
__global__ void __launch_bounds__(128) quantize_by_warp_kernel(const T* __restrict__ x, long long ld_x, int8_t* __restrict__ q, long long ld_q,
                                                               float* __restrict__ scale, long long M, int K) {
    constexpr int N = Vec16<T>::kN;
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31;
    const long long row0 = (static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5)) * R;
    if (row0 >= M) return;
    const int rows = static_cast<int>(min(static_cast<long long>(R), M - row0));
    uint4 v[R][NV];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (lane + i * 32) * N;
            v[r][i] = k < K && r < rows ? *reinterpret_cast<const uint4*>(x + (row0 + r) * ld_x + k) : make_uint4(0, 0, 0, 0);
        }
    uint32_t mine = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) top = max(top, top_of<T>(v[r][i]));
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane % R == r) mine = top;
    }
    const float my_scale = i8_scale(mine), my_inv = i8_inverse(my_scale);
    if (lane < rows) scale[row0 + lane] = my_scale;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float s = __shfl_sync(0xffffffffu, my_scale, r), inv = __shfl_sync(0xffffffffu, my_inv, r);
        if (r >= rows) break;
        int8_t* qr = q + (row0 + r) * ld_q;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int k = (lane + i * 32) * N;
            if (k >= K) continue;
            uint32_t w[N / 4];
            quantize_vec<T>(v[r][i], s, inv, w);
            if constexpr (N == 4) *reinterpret_cast<uint32_t*>(qr + k) = w[0];
            else *reinterpret_cast<uint2*>(qr + k) = make_uint2(w[0], w[1]);
        }
    }
}
// longer rows: a block of THREADS threads per row.
template <typename T, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS) quantize_by_block_kernel(const T* __restrict__ x, long long ld_x, int8_t* __restrict__ q, long long ld_q,
                                                                    float* __restrict__ scale, int K) {
    constexpr int N = Vec16<T>::kN;
    __shared__ uint32_t part[THREADS / 32];
    pdl_wait();
    pdl_launch_dependents();
    const long long row = blockIdx.x;
    const T* xr = x + row * ld_x;
    uint4 v[NV];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (static_cast<int>(threadIdx.x) + i * THREADS) * N;
        v[i] = k < K ? *reinterpret_cast<const uint4*>(xr + k) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) top = max(top, top_of<T>(v[i]));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) top = max(top, part[i]);
    const float s = i8_scale(top), inv = i8_inverse(s);
    int8_t* qr = q + row * ld_q;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int k = (static_cast<int>(threadIdx.x) + i * THREADS) * N;
        if (k >= K) continue;
        uint32_t w[N / 4];
        quantize_vec<T>(v[i], s, inv, w);
        if constexpr (N == 4) *reinterpret_cast<uint32_t*>(qr + k) = w[0];
        else *reinterpret_cast<uint2*>(qr + k) = make_uint2(w[0], w[1]);
    }
    if (threadIdx.x == 0) scale[row] = s;
}

// Any length, any alignment: one block per row, value by value; the second pass over the row comes from L1 / L2.  Bound by its narrow
// loads: 1.1 TB/s in bf16 and 1.8 in fp32 at K = 4001 (6.8 at 4000), 1.8 in fp32 at K = 12288.
template <typename T>
__global__ void __launch_bounds__(512) quantize_any_kernel(const T* __restrict__ x, long long ld_x, int8_t* __restrict__ q, long long ld_q,
                                                           float* __restrict__ scale, int K) {
    __shared__ uint32_t part[16];
    pdl_wait();
    pdl_launch_dependents();
    const long long row = blockIdx.x;
    const T* xr = x + row * ld_x;
    uint32_t top = 0;
#pragma unroll 4
    for (int k = threadIdx.x; k < K; k += blockDim.x) top = max(top, magnitude_bits(to_f32(xr[k])));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const float s = i8_scale(__reduce_max_sync(0xffffffffu, lane < static_cast<int>(blockDim.x >> 5) ? part[lane] : 0u));
    int8_t* qr = q + row * ld_q;
#pragma unroll 4
    for (int k = threadIdx.x; k < K; k += blockDim.x) qr[k] = static_cast<int8_t>(i8_quantize(to_f32(xr[k]), s));
    if (threadIdx.x == 0) scale[row] = s;
}

template <typename T>
int launch_quantize_t(const T* x, long long ld_x, int8_t* q, long long ld_q, float* scale, long long rows, int K, cudaStream_t st) {
    constexpr int N = Vec16<T>::kN;
    const bool vec = (reinterpret_cast<uintptr_t>(x) | (ld_x * sizeof(T))) % 16 == 0 && (reinterpret_cast<uintptr_t>(q) | ld_q) % N == 0 && K % N == 0;
    const int pieces = (K + N - 1) / N;
    // Many rows: small blocks with as much in flight per thread as fits (16384 x 4096 bf16 31.4 us, 6.4 TB/s, against 36.6 with 256
    // threads of two pieces; 65536 x 256 bf16 10.5 against 17.6 with one row per warp); few: all of a row at once (48 x 4096
    // 1.6 us against 2.2).
    const bool many = rows >= 32ll * num_sms();
    cudaError_t e;
#define PPML_W(NV, R) launch_pdl(quantize_by_warp_kernel<T, NV, R>, dim3(static_cast<unsigned>((rows + 4 * R - 1) / (4 * R))), dim3(128), 0, st, x, ld_x, q, ld_q, scale, rows, K)
#define PPML_B(THREADS, NV) launch_pdl(quantize_by_block_kernel<T, THREADS, NV>, dim3(static_cast<unsigned>(rows)), dim3(THREADS), 0, st, x, ld_x, q, ld_q, scale, K)
    if (!vec || pieces > 2048) e = launch_pdl(quantize_any_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(K <= 1024 ? 128 : 512), 0, st, x, ld_x, q, ld_q, scale, K);
    else if (pieces <= 32) e = many ? PPML_W(1, 4) : PPML_W(1, 1);
    else if (pieces <= 64) e = many ? PPML_W(2, 2) : PPML_W(2, 1);
    else if (pieces <= 128) e = PPML_W(4, 1);
    else if (pieces <= 256) e = many ? PPML_B(64, 4) : PPML_B(256, 1);
    else if (pieces <= 512) e = many ? PPML_B(64, 8) : PPML_B(256, 2);
    else if (pieces <= 1024) e = many ? PPML_B(128, 8) : PPML_B(256, 4);
    else e = PPML_B(512, 4);
#undef PPML_W
#undef PPML_B
    if (e != cudaSuccess) { cudaGetLastError(); return ST_LAUNCH; }
    return ST_OK;
}

// 64 x 64 outputs per block of 256 threads, 4 x 4 each; 64 k per step as 16 words of four, dp4a.  Rows that are not 4-byte
// aligned are read byte by byte.
constexpr int kT = 64, kWords = 16;

__device__ __forceinline__ int load_word(const int8_t* row, int k, int K, bool aligned) {
    if (aligned && k + 4 <= K) return *reinterpret_cast<const int*>(row + k);
    uint32_t v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (k + i < K) v |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * i);
    return static_cast<int>(v);
}

template <typename T>
__global__ void __launch_bounds__(256) i8_dp4a_kernel(I8Product p) {
    __shared__ int As[kWords][kT + 1], Bs[kWords][kT + 1];
    const long long m0 = static_cast<long long>(blockIdx.x) * kT, n0 = static_cast<long long>(blockIdx.y) * kT;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const bool a_al = ((reinterpret_cast<uintptr_t>(p.A) | p.lda) & 3) == 0, b_al = ((reinterpret_cast<uintptr_t>(p.B) | p.ldb) & 3) == 0;
    int acc[4][4] = {};
    for (int k0 = 0; k0 < p.K; k0 += 4 * kWords) {
        for (int i = threadIdx.x; i < kT * kWords; i += 256) {
            const int w = i & (kWords - 1), r = i >> 4;
            As[w][r] = m0 + r < p.M ? load_word(p.A + (m0 + r) * p.lda, k0 + 4 * w, p.K, a_al) : 0;
            Bs[w][r] = n0 + r < p.N ? load_word(p.B + (n0 + r) * p.ldb, k0 + 4 * w, p.K, b_al) : 0;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            int a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { a[i] = As[w][ty + 16 * i]; b[i] = Bs[w][tx + 16 * i]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __dp4a(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long m = m0 + ty + 16 * i;
        if (m >= p.M) continue;
        const float sa = p.a_scale[m];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const long long n = n0 + tx + 16 * j;
            if (n >= p.N) continue;
            float y = i8_epilogue(acc[i][j], sa, p.b_scale[n], p.bias ? p.bias[n] : 0.0f, p);
            if (p.gate) y *= to_f32(static_cast<const T*>(p.gate)[m * p.ld_gate + n]);
            static_cast<T*>(p.C)[m * p.ldc + n] = from_f32<T>(y);
        }
    }
}

}  // namespace

int launch_quantize_tokens(const void* x, int type, long long ld_x, int8_t* q, long long ld_q, float* scale, long long rows, int K,
                           cudaStream_t st) {
    switch (type) {
        case kTypeF32: return launch_quantize_t(static_cast<const float*>(x), ld_x, q, ld_q, scale, rows, K, st);
        case kTypeF16: return launch_quantize_t(static_cast<const __half*>(x), ld_x, q, ld_q, scale, rows, K, st);
        default: return launch_quantize_t(static_cast<const __nv_bfloat16*>(x), ld_x, q, ld_q, scale, rows, K, st);
    }
}

int launch_i8_dp4a(const I8Product& p, cudaStream_t st) {
    const dim3 grid(static_cast<unsigned>((p.M + static_cast<long long>(kT) - 1) / kT), static_cast<unsigned>((p.N + static_cast<long long>(kT) - 1) / kT));
    if ((p.N + static_cast<long long>(kT) - 1) / kT > 65535) return ST_TOO_LARGE;
    switch (p.c_type) {
        case kTypeF32: i8_dp4a_kernel<float><<<grid, 256, 0, st>>>(p); break;
        case kTypeF16: i8_dp4a_kernel<__half><<<grid, 256, 0, st>>>(p); break;
        default: i8_dp4a_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
    }
    return cudaGetLastError() == cudaSuccess ? ST_OK : ST_LAUNCH;
}

}  // namespace ppml_b200
