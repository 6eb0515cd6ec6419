// umma_i8.cu -- C[token][channel] = epilogue(sum_k A[token][k] * W[channel][k]) in 8-bit integers on tcgen05 (kind::i8).
//
// The weights are the tensor core's M operand and the tokens its N operand: the accumulator then holds a channel per TMEM lane
// and a token per column, a warp that reads one column holds 32 neighbouring channels of one token, and the results leave the
// registers as whole coalesced pieces of a row of C, whatever its pitch and type.  The whole sum over K stays in int32 in
// TMEM, so splitting K changes nothing; each output sees one epilogue.
//
// Both operands are K-major int8 tiles of 128 bytes of K per stage (128-byte swizzle), pulled in by TMA; rows and K beyond the
// tensors read as zeros.  Warp 0 = TMA, warp 1 = MMA issue and TMEM owner, warps 2 - 17 = epilogue (four per TMEM lane quarter).
//
// What bounds it: with a long K the tensor pipe (16384 x 4096 -> 8192 335 us, 3.28 PFLOP/s, twice what cuBLAS reaches in bf16; back to
// back the power limit takes it to some 400), with a short one the results' way out: 65536 x 256 -> 512 fp32 27 us (5.6 TB/s),
// -> 1024 bf16 36 us (4.2 TB/s: issue of the epilogue, a third of it conversions), with SiLU 52 us (two transcendental instructions
// an output are 30 us alone); with few tokens the weights' way in: 48 x 4096 -> 8192 10.4 us cold (3.3 TB/s over 128 CTAs).
#include <atomic>

#include "i8_common.cuh"
#include "tma_host.h"

namespace ppml_b200 {
namespace {

constexpr int kFirstEpi = 2, kEpiWarps = 16, kEpiParts = kEpiWarps / 4;
constexpr int kThreadsI8 = 32 * (kFirstEpi + kEpiWarps);
constexpr int kMaxStages = 8;
constexpr int kSmemMax = 227 * 1024;
constexpr int kRowsA = 128;                        // channels per CTA
constexpr int kABytes = kRowsA * 128;
constexpr int kBarBytes = 256, kScaleBytes = kEpiWarps * 32 * 4;

struct I8Tc {
    I8Product p;
    int bn;                                        // tokens per tile (the MMA's N): a multiple of 16 (pairs: of 32), at most 256
    int stages, stage_bytes;
    int tiles_n, tiles_t, kblocks;
    int tmem_cols;                                 // power of two >= what the accumulators take
    int* err;
};

// ---- cluster helpers ----
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t map_to(uint32_t saddr, uint32_t rank) {
    uint32_t r; asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank)); return r;
}
__device__ __forceinline__ void cluster_sync_all() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Orders nothing but the tensor memory reads that tcgen05.fence::before_thread_sync put before it: a release at cluster scope
// would make the warp wait for its stores of results every time (it took a third of the epilogue).
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_s32(uint32_t cluster_addr) {
    uint32_t v; asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory"); return v;
}

// ---- the forms that a pair of CTAs uses ----
template <int CG> __device__ __forceinline__ void tmem_alloc_cg(uint32_t dst, uint32_t n) {
    if constexpr (CG == 1) tmem_alloc(dst, n);
    else asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(n) : "memory");
}
template <int CG> __device__ __forceinline__ void tmem_free_cg(uint32_t taddr, uint32_t n) {
    if constexpr (CG == 1) { tmem_relinquish(); tmem_dealloc(taddr, n); }
    else {
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(n) : "memory");
    }
}
// CG = 2: into this CTA's shared memory, counted on a barrier of the pair's leader
template <int CG> __device__ __forceinline__ void load_tile(uint32_t dst, const void* tm, uint32_t bar, int x, int y) {
    if constexpr (CG == 1) tma_load_3d(dst, tm, bar, x, y, 0);
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];"
            ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y), "r"(0) : "memory");
}
template <int CG> __device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    if constexpr (CG == 1) umma<MmaKind::I8>(d, a, b, idesc, acc);
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
// arrives on the barrier at this offset in every CTA of the group once all MMAs issued so far are done
template <int CG> __device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (CG == 1) umma_commit(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}

// One stage: up to four MMAs of 32 k and the commit that hands the stage back.  The whole warp walks the loops around this with
// uniform values and one elected lane issues: descriptors then stay in uniform registers (inside a branch taken by lane 0
// alone, the four MMAs took 540 cycles to issue, longer than the 512 they run).
template <int CG>
__device__ __forceinline__ void issue_block(bool lead, uint32_t d, uint64_t desc_a, uint32_t idesc, int steps, uint32_t accumulate, uint32_t empty) {
    const uint64_t desc_b = desc_a + (kABytes >> 4);
    if (lead) {
        if (steps == 4) {
            mma_i8<CG>(d, desc_a, desc_b, idesc, accumulate);
            mma_i8<CG>(d, desc_a + 2, desc_b + 2, idesc, 1u);
            mma_i8<CG>(d, desc_a + 4, desc_b + 4, idesc, 1u);
            mma_i8<CG>(d, desc_a + 6, desc_b + 6, idesc, 1u);
        } else {
            for (int k = 0; k < steps; ++k) mma_i8<CG>(d, desc_a + 2 * k, desc_b + 2 * k, idesc, k == 0 ? accumulate : 1u);
        }
        commit<CG>(empty);
    }
    __syncwarp();
}

// ---- epilogue of 32 tokens x this lane's channel ----
// Gates of 32 tokens, requested before their sums are there.
template <typename T, int MORE> struct Gates {
    uint32_t w[MORE < 2 ? 1 : sizeof(T) == 2 ? 16 : 32];
    __device__ __forceinline__ void load(const I8Product& p, long long t0, int left, long long n) {
        if (MORE < 2 || n >= p.N) return;
        const T* g = static_cast<const T*>(p.gate) + t0 * p.ld_gate + n;
#pragma unroll
        for (int j = 0; j < 32; ++j, g += p.ld_gate) {
            if constexpr (sizeof(T) == 4) {
                w[j] = j < left ? *reinterpret_cast<const uint32_t*>(g) : 0u;
            } else {
                const uint32_t v = j < left ? *reinterpret_cast<const uint16_t*>(g) : 0u;
                w[j / 2] = j & 1 ? w[j / 2] | v << 16 : v;
            }
        }
    }
    __device__ __forceinline__ float at(int j) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
        else { const uint16_t v = static_cast<uint16_t>(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu); return to_f32(*reinterpret_cast<const T*>(&v)); }
    }
};

// Columns of TMEM in eights, enough for `left` (1 to 32) tokens; the rest of r stays undefined.  Each way waits for itself: until
// then nothing may touch the registers, a move where the ways meet included.
__device__ __forceinline__ void load_sums8(uint32_t at, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_sums(uint32_t at, int left, uint32_t (&r)[32]) {
    if (left > 24) { tmem_ld32(at, r); tmem_ld_wait(); }
    else if (left > 16) { load_sums8(at, r); load_sums8(at + 8, r + 8); load_sums8(at + 16, r + 16); tmem_ld_wait(); }
    else if (left > 8) { load_sums8(at, r); load_sums8(at + 8, r + 8); tmem_ld_wait(); }
    else { load_sums8(at, r); tmem_ld_wait(); }
}

// an activation's number as a type
template <int V> struct Kind { static constexpr int value = V; };

// The sums of `left` tokens (>= 32: all) from t0 on in this lane's channel n become results and go to C, eight tokens at a time.
// MORE: 0 nothing follows, 1 an activation, 2 a gate (and perhaps an activation): instances of their own, because the registers of the
// gates and the code of the activations cost the plain ones a fifth of their time.  16-bit results in rows on 4 bytes go
// out two channels a lane: neighbouring lanes exchange one of two tokens, an even lane keeps its first token and takes the
// neighbour's, an odd one the second.
template <typename T, int MORE>
__device__ __forceinline__ void finish_chunk(const I8Product& p, const uint32_t (&sum)[32], const Gates<T, MORE>& gate, float* scale_buf, float scale,
                                             long long t0, int left, long long n, float b_scale, float bias, int lane) {
    __syncwarp();
    scale_buf[lane] = scale;
    __syncwarp();
    const uint64_t b2 = pack2(b_scale, b_scale), bias2 = pack2(bias, bias);
    T* c = static_cast<T*>(p.C) + t0 * p.ldc + n;
    const uint64_t ldc = static_cast<uint32_t>(p.ldc);         // below 2^32 (the launcher's condition): one multiply-add per address
    auto results = [&](int j0, float (&y)[8], auto kind) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) {
            const float4 s = reinterpret_cast<const float4*>(scale_buf)[(j0 + j) / 4];
            auto f = [&](int i) { return static_cast<float>(static_cast<int>(sum[j0 + j + i])); };
            unpack2(ffma2(fmul2(pack2(f(0), f(1)), pack2(s.x, s.y)), b2, bias2), y[j], y[j + 1]);
            unpack2(ffma2(fmul2(pack2(f(2), f(3)), pack2(s.z, s.w)), b2, bias2), y[j + 2], y[j + 3]);
        }
        if constexpr (MORE > 0) i8_act_all(kind.value, y);
        if constexpr (MORE == 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= gate.at(j0 + j);
        }
    };
    const bool odd = lane & 1;
    uint32_t* to = reinterpret_cast<uint32_t*>(c + (odd ? ldc - 1 : 0));       // two channels of one token
    const uint32_t pick = odd ? 0x3276 : 0x5410;
    auto store_paired = [&](int j0, const float (&y)[8]) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint32_t own = narrow2(y[j], y[j + 1], T()), other = __shfl_xor_sync(0xffffffffu, own, 1);
                to[ldc / 2 * (j0 + j)] = __byte_perm(own, other, pick);
            }
        }
    };
    auto store = [&](int j0, const float (&y)[8], bool all) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (all || j0 + j < left) c[ldc * (j0 + j)] = from_f32<T>(y[j]);
    };
    const bool paired = sizeof(T) == 2 && n - lane + 32 <= p.N && ((reinterpret_cast<uintptr_t>(p.C) >> 1 | p.ldc) & 1) == 0;
    // Each loop has one kind of store, and no masks on a whole chunk: 65536 x 256 -> 256 fp32 sigmoid 22.2 -> 19.6 us; 65536 x 256 -> 1024
    // bf16 GELU 85 us with both kinds of stores behind a branch, 72; 1999 x 1000 -> 777 fp16 SiLU and gate 8.5 and 8.1.
    auto run = [&](auto kind) {
        if (left >= 32 && paired) {
#pragma unroll
            for (int j0 = 0; j0 < 32; j0 += 8) { float y[8]; results(j0, y, kind); store_paired(j0, y); }
        } else if (n < p.N) {
            if ((MORE == 0 || sizeof(T) == 4) && left >= 32) {     // 16 bits with an activation: one copy of it less
#pragma unroll
                for (int j0 = 0; j0 < 32; j0 += 8) { float y[8]; results(j0, y, kind); store(j0, y, true); }
            } else {
#pragma unroll
                for (int j0 = 0; j0 < 32; j0 += 8)
                    if (j0 < left) { float y[8]; results(j0, y, kind); store(j0, y, false); }
            }
        }
    };
    if constexpr (MORE == 0) {
        run(Kind<0>());
    } else {                                       // the kind known to the loops: 65536 x 256 -> 1024 bf16 SiLU 60 -> 52 us, GELU 71 -> 58
        switch (p.act) {
            case 0: run(Kind<0>()); break;
            case 1: run(Kind<1>()); break;
            case 2: run(Kind<2>()); break;
            case 3: run(Kind<3>()); break;
            case 4: run(Kind<4>()); break;
            default: run(Kind<5>());
        }
    }
    __syncwarp();
}

// On an abort the copies that are still on their way must not land in the shared memory of a later block.
__device__ __noinline__ void wait_for_copies() {
    const long long t0 = clock64();
    while (clock64() - t0 < 4000000LL) __nanosleep(1000);
}

// Persistent: a CTA (CG = 1) or a pair of CTAs (CG = 2: 256 channels, each CTA holding half of the weight rows and half of the
// token rows of a stage) takes every gridDim-th tile; two accumulators in TMEM, so that a tile's epilogue runs under the
// next tile's MMAs.
template <typename T, int CG, int MORE>
__global__ void __launch_bounds__(kThreadsI8, 1)
i8_tiles_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA, const I8Tc q) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];      // no static shared memory: it starts on the swizzle's 1024 bytes
    const uint32_t base = smem_u32(smem_raw);
    uint8_t* gen = smem_raw;
    const uint32_t bars = base + q.stages * q.stage_bytes;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (kMaxStages + s); };
    auto tfull = [&](int a) { return bars + 8u * (2 * kMaxStages + a); };
    auto tempty = [&](int a) { return bars + 8u * (2 * kMaxStages + 2 + a); };
    uint8_t* tail = gen + q.stages * q.stage_bytes;
    volatile int* cta_abort = reinterpret_cast<volatile int*>(tail + 8 * (2 * kMaxStages + 4));
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 8 * (2 * kMaxStages + 4) + 8);
    float* scales = reinterpret_cast<float*>(tail + kBarBytes);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
    const int group = blockIdx.x / CG, groups = gridDim.x / CG;
    const int tiles = q.tiles_n * q.tiles_t;

    if (threadIdx.x == 0) {
        prefetch_tmap(&tmW); prefetch_tmap(&tmA);
        for (int s = 0; s < q.stages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        for (int a = 0; a < 2; ++a) { mbar_init(tfull(a), 1); mbar_init(tempty(a), CG * kEpiWarps); }
        *cta_abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc_cg<CG>(smem_u32(tmem_slot), q.tmem_cols);
    tc_fence_before();
    __syncthreads();
    if (CG == 2) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    // tile index -> (channel tile, token tile): eight token tiles side by side, so that tiles in flight share operands in L2
    auto tile_at = [&](int i, int& tn, int& tt) {
        const int per = 8 * q.tiles_n, g = i / per, first = g * 8, r = i - g * per;
        const int width = min(8, q.tiles_t - first);
        tn = r / width; tt = first + r - tn * width;
    };
    const int b_rows = q.bn / CG;

    if (warp == 0) {
        if (lane == 0) {
            int s = 0; uint32_t ph = 0; bool ok = true;
            int issued = 0;
            for (int i = group; i < tiles && ok; i += groups) {
                int tn, tt; tile_at(i, tn, tt);
                const int yw = tn * kRowsA * CG + static_cast<int>(rank) * kRowsA;
                const int ya = tt * q.bn + static_cast<int>(rank) * b_rows;
                for (int kb = 0; kb < q.kblocks; ++kb) {
                    if (!mbar_wait(empty(s), ph ^ 1u, cta_abort, q.err, 0x800 | s)) { ok = false; break; }
                    const uint32_t at = base + s * q.stage_bytes;
                    const uint32_t bar = CG == 2 ? map_to(full(s), 0) : full(s);
                    if (rank == 0) mbar_arrive_expect_tx(full(s), static_cast<uint32_t>(CG * q.stage_bytes));
                    load_tile<CG>(at, &tmW, bar, kb * 128, yw);
                    load_tile<CG>(at + kABytes, &tmA, bar, kb * 128, ya);
                    ++issued;
                    if (++s == q.stages) { s = 0; ph ^= 1u; }
                }
            }
            // every stage has been handed back before this CTA may leave: commits of the pair still arrive here
            for (int n = min(issued, q.stages); n > 0 && ok; --n) {
                if (issued < q.stages && n == issued) { s = 0; ph = 1u; }      // fewer loads than stages: the first ones, phase 0
                ok = mbar_wait(empty(s), ph ^ 1u, cta_abort, q.err, 0x810 | s);
                if (++s == q.stages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t idesc = make_idesc(2, 1, 1, 0, 0, kRowsA * CG, q.bn);
            const int last_steps = (q.p.K - (q.kblocks - 1) * 128 + 31) / 32;
            const uint64_t desc0 = make_smem_desc(base, 16, 1024, kLayoutSW128);
            const uint32_t step = static_cast<uint32_t>(q.stage_bytes) >> 4;
            const bool lead = elect_one();
            int s = 0; uint32_t ph = 0; bool ok = true; int acc = 0; uint32_t aph = 0;
            for (int i = group; i < tiles && ok; i += groups) {
                if (!__all_sync(0xffffffffu, mbar_wait(tempty(acc), aph ^ 1u, cta_abort, q.err, 0x820 | acc))) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * (q.tmem_cols / 2);
                for (int kb = 0; kb < q.kblocks; ++kb) {
                    if (!__all_sync(0xffffffffu, mbar_wait(full(s), ph, cta_abort, q.err, 0x830 | s))) { ok = false; break; }
                    tc_fence_after();
                    issue_block<CG>(lead, d, desc0 + static_cast<uint64_t>(s * step), idesc, kb == q.kblocks - 1 ? last_steps : 4, kb != 0, empty(s));
                    if (++s == q.stages) { s = 0; ph ^= 1u; }
                }
                if (!ok) break;
                if (lead) commit<CG>(tfull(acc));
                __syncwarp();
                if (++acc == 2) { acc = 0; aph ^= 1u; }
            }
        }
    } else {
        const int quarter = warp & 3, part = (warp - kFirstEpi) >> 2;
        float* scale_buf = scales + (warp - kFirstEpi) * 32;
        int acc = 0; uint32_t aph = 0;
        for (int i = group; i < tiles; i += groups) {
            int tn, tt; tile_at(i, tn, tt);
            const long long n = static_cast<long long>(tn) * kRowsA * CG + rank * kRowsA + quarter * 32 + lane;
            const bool n_ok = n < q.p.N;
            const float bs = n_ok ? q.p.b_scale[n] : 0.0f, bias = n_ok && q.p.bias ? q.p.bias[n] : 0.0f;
            const long long t0 = static_cast<long long>(tt) * q.bn;
            const long long rest = q.p.M - t0;
            const int cols = static_cast<int>(rest < q.bn ? rest : q.bn);
            // This warp's tokens of the tile: a fourth, in chunks of 32 at most.  Where an activation follows the fourth is counted in
            // eights (48 x 1024 -> 4096 GELU: 6.0 us in whole chunks, 5.0), else in whole chunks, which need no masks (65536 x 256 ->
            // 256 bf16 12.8 us, 13.7 in eights).
            constexpr int kGrain = MORE > 0 ? 8 : 32;
            const int share = (cols + kGrain * kEpiParts - 1) / (kGrain * kEpiParts) * kGrain, first = part * share, mine = min(share, cols - first);
            float scale[2];                        // of the chunks this warp will read, requested before the wait
            Gates<T, MORE> gate;
#pragma unroll
            for (int k = 0; k < 2; ++k) scale[k] = lane + 32 * k < mine ? q.p.a_scale[t0 + first + 32 * k + lane] : 0.0f;
            gate.load(q.p, t0 + first, min(mine, 32), n);
            if (!__all_sync(0xffffffffu, mbar_wait(tfull(acc), aph, cta_abort, q.err, 0x840 | acc))) break;
            tc_fence_after();
            const uint32_t d = tmem + acc * (q.tmem_cols / 2) + (static_cast<uint32_t>(quarter * 32) << 16) + first;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int left = min(32, mine - 32 * k);
                uint32_t r[32];
                if (left > 0) {
                    if (k == 1) gate.load(q.p, t0 + first + 32, left, n);
                    __syncwarp();
                    load_sums(d + 32 * k, left, r);
                }
                // the last read of this warp, or none in this tile: the accumulator may be written again
                if (k == (mine > 32 ? 1 : 0)) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) { if (CG == 2) mbar_arrive_cluster(map_to(tempty(acc), 0)); else mbar_arrive(tempty(acc)); }
                }
                if (left > 0) finish_chunk<T, MORE>(q.p, r, gate, scale_buf, scale[k], t0 + first + 32 * k, left, n, bs, bias, lane);
            }
            if (++acc == 2) { acc = 0; aph ^= 1u; }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*cta_abort && threadIdx.x == 0) wait_for_copies();
    __syncwarp();
    if (CG == 2) cluster_sync_all();
    tc_fence_after();
    if (warp == 1) tmem_free_cg<CG>(tmem, q.tmem_cols);
}

// Few tiles and a long K: one tile per cluster of `parts` CTAs (2, 4, 8), each of which sums its share of K; the int32 partial sums
// meet in shared memory, every CTA finishing its share of the tokens.
template <typename T, int MORE>
__global__ void __launch_bounds__(kThreadsI8, 1)
i8_parts_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA, const I8Tc q, const int parts) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];      // no static shared memory: it starts on the swizzle's 1024 bytes
    const uint32_t base = smem_u32(smem_raw);
    uint8_t* gen = smem_raw;
    const uint32_t bars = base + q.stages * q.stage_bytes;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (kMaxStages + s); };
    const uint32_t tfull = bars + 8u * 2 * kMaxStages;
    uint8_t* tail = gen + q.stages * q.stage_bytes;
    volatile int* cta_abort = reinterpret_cast<volatile int*>(tail + 8 * (2 * kMaxStages + 4));
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 8 * (2 * kMaxStages + 4) + 8);
    float* scales = reinterpret_cast<float*>(tail + kBarBytes);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(cluster_rank());
    const int tile = blockIdx.x / parts, tn = tile / q.tiles_t, tt = tile - tn * q.tiles_t;
    const int kb0 = static_cast<int>(static_cast<long long>(q.kblocks) * rank / parts);
    const int kb1 = static_cast<int>(static_cast<long long>(q.kblocks) * (rank + 1) / parts);

    if (threadIdx.x == 0) {
        prefetch_tmap(&tmW); prefetch_tmap(&tmA);
        for (int s = 0; s < q.stages; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
        mbar_init(tfull, 1);
        *cta_abort = 0;
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), q.tmem_cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    const long long t0 = static_cast<long long>(tt) * q.bn;
    const long long rest = q.p.M - t0;
    const int cols = static_cast<int>(rest < q.bn ? rest : q.bn);
    if (warp == 0) {
        if (lane == 0) {
            int s = 0; uint32_t ph = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait(empty(s), ph ^ 1u, cta_abort, q.err, 0x900 | s)) break;
                const uint32_t at = base + s * q.stage_bytes;
                mbar_arrive_expect_tx(full(s), static_cast<uint32_t>(q.stage_bytes));
                load_tile<1>(at, &tmW, full(s), kb * 128, tn * kRowsA);
                load_tile<1>(at + kABytes, &tmA, full(s), kb * 128, static_cast<int>(t0));
                if (++s == q.stages) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        const uint32_t idesc = make_idesc(2, 1, 1, 0, 0, kRowsA, q.bn);
        const int last_steps = (q.p.K - (q.kblocks - 1) * 128 + 31) / 32;
        const uint64_t desc0 = make_smem_desc(base, 16, 1024, kLayoutSW128);
        const uint32_t step = static_cast<uint32_t>(q.stage_bytes) >> 4;
        const bool lead = elect_one();
        int s = 0; uint32_t ph = 0; bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!__all_sync(0xffffffffu, mbar_wait(full(s), ph, cta_abort, q.err, 0x930 | s))) { ok = false; break; }
            tc_fence_after();
            issue_block<1>(lead, tmem, desc0 + static_cast<uint64_t>(s * step), idesc, kb == q.kblocks - 1 ? last_steps : 4, kb != kb0, empty(s));
            if (++s == q.stages) { s = 0; ph ^= 1u; }
        }
        if (ok && lead) umma_commit(tfull);
    }
    __syncwarp();
    const int quarter = warp & 3, part = (warp - kFirstEpi) >> 2;
    const long long n = static_cast<long long>(tn) * kRowsA + quarter * 32 + lane;
    const bool n_ok = n < q.p.N;
    const float bs = n_ok ? q.p.b_scale[n] : 0.0f, bias = n_ok && q.p.bias ? q.p.bias[n] : 0.0f;
    float* scale_buf = scales + (warp - kFirstEpi) * 32;
    if (warp >= kFirstEpi) {
        if (__all_sync(0xffffffffu, mbar_wait(tfull, 0, cta_abort, q.err, 0x940))) {
            tc_fence_after();
            // a fourth of the tile's tokens in eights: 32 at most, since bn <= 128
            const int share = (cols + 8 * kEpiParts - 1) / (8 * kEpiParts) * 8, c = part * share, left = min(share, cols - c);
            if (left > 0) {
                uint32_t r[32];
                __syncwarp();
                load_sums(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + c, left, r);
                // the stages are free: every load has landed and every MMA has read
                uint32_t* buf = reinterpret_cast<uint32_t*>(gen) + c * kRowsA + quarter * 32 + lane;
#pragma unroll
                for (int j0 = 0; j0 < 32; j0 += 8)
                    if (j0 < left) {
#pragma unroll
                        for (int j = j0; j < j0 + 8; ++j) buf[j * kRowsA] = r[j];
                    }
            }
        }
    }
    __syncwarp();
    cluster_sync_all();
    if (warp >= kFirstEpi) {
        // tokens in chunks of 8, dealt to the CTAs and within a CTA to its four groups of warps
        for (int c = (rank + part * parts) * 8; c < cols; c += 8 * parts * kEpiParts) {
            uint32_t v[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0;
            const int left = min(8, cols - c);
            const float s = lane < left ? q.p.a_scale[t0 + c + lane] : 0.0f;
            Gates<T, MORE> gate;
            gate.load(q.p, t0 + c, left, n);
            const uint32_t at = base + static_cast<uint32_t>((c * kRowsA + quarter * 32 + lane) * 4);
            for (int r = 0; r < parts; ++r) {
                const uint32_t there = map_to(at, static_cast<uint32_t>((rank + r) % parts));
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += ld_cluster_s32(there + j * kRowsA * 4);
            }
            finish_chunk<T, MORE>(q.p, v, gate, scale_buf, s, t0 + c, left, n, bs, bias, lane);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*cta_abort && threadIdx.x == 0) wait_for_copies();
    __syncwarp();
    cluster_sync_all();
    tc_fence_after();
    if (warp == 1) { tmem_relinquish(); tmem_dealloc(tmem, q.tmem_cols); }
}

int pow2_at_least(int v, int lo) { int c = lo; while (c < v) c *= 2; return c; }

template <auto kernel, typename... Args>
cudaError_t launch_cluster(int grid, int cluster, size_t smem, cudaStream_t st, const Args&... args) {
    // the attribute once per kernel and device (two threads may both set it)
    static std::atomic<uint64_t> allowed{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax);
        if (e != cudaSuccess) return e;
        allowed.fetch_or(bit, std::memory_order_relaxed);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid); cfg.blockDim = dim3(kThreadsI8); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster; attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// How a product is cut: `pair` 1 persistent single CTAs, 2 persistent pairs, 0 one tile per cluster of `parts` CTAs.
struct Plan { int pair = 1, bn = 256, parts = 1; };

// The cut with the shortest estimate, in cycles, for the busiest CTA.  A stage of 128 k takes 2.1 cycles a row (the rate at which
// tiles come out of L2: a pair fetches half of the token rows each), a tile's epilogue 8 a token, a tile 400 besides, a pair's
// hand-shakes 800; parts of K cost 1300 + 30 a token for the partial sums' way through shared memory, and a B200 holds at once only as
// many clusters of 2, 4 and 8 CTAs as kClustersHeld says.  Over 70 sizes of 1 to 8192 tokens the cut so chosen is 1.2 % slower than the
// fastest one in the mean (17 % at most); without kClustersHeld it was 84 % at 1 x 4096 -> 2048 (9.7 for 5.3 us).  Best
// against other cuts (us, bf16 results): 408 x 1024 -> 1024 32 tokens a tile 4.5, 128 in four parts 6.8; 200 x 8192 -> 1024 64 in four
// parts 9.2, 32 in two 11.6; 1999 x 1000 -> 777 96 6.4, 128 6.9; 8192 x 256 -> 512 single 5.4, pairs 6.2; 5000 x 4000 -> 1000
// pairs 24.4, single 30.6; 65536 x 256 -> 256 tiles of 256 13.5, of 128 14.5.
constexpr int kClustersHeld[9] = {0, 148, 74, 0, 33, 0, 0, 0, 15};     // one CTA an SM, cudaOccupancyMaxActiveClusters

Plan choose_anew(const I8Product& p) {
    const long long sms = num_sms(), kb = (p.K + 127) / 128, M = p.M;
    Plan best;
    long long least = INT64_MAX;
    auto consider = [&](Plan plan) {
        const int cg = plan.pair == 2 ? 2 : 1;
        const long long tn = (p.N + 128ll * cg - 1) / (128 * cg), tt = (M + plan.bn - 1) / plan.bn, units = tn * tt;
        const long long at_once = plan.pair == 0 ? kClustersHeld[plan.parts] : sms / cg;
        const long long rounds = (units + at_once - 1) / at_once, steps = (kb + plan.parts - 1) / plan.parts;
        const long long fill = steps * (128 + plan.bn / cg) * 21 / 10;
        const long long cost = rounds * (fill + (plan.pair == 0 ? 1300 + 30 * plan.bn : 8 * plan.bn + 400 + (cg == 2 ? 800 : 0)));
        if (cost < least) { least = cost; best = plan; }
    };
    const int most = M >= 256 ? 256 : static_cast<int>((M + 15) / 16 * 16);        // whole tiles of tokens for small M
    for (int bn = most < 32 ? most : 32; bn <= most; bn += bn < 32 ? 16 : 32) {
        consider({1, bn, 1});
        if (p.N > 128 && bn >= 64) consider({2, bn, 1});
        if (bn <= 128)
            for (int parts = 2; parts <= 8 && 2 * parts <= kb; parts *= 2) consider({0, bn, parts});
    }
    if (most > 32 && most % 32 != 0) {             // one tile of exactly M tokens
        consider({1, most, 1});
        if (most <= 128)
            for (int parts = 2; parts <= 8 && 2 * parts <= kb; parts *= 2) consider({0, most, parts});
    }
    return best;
}

// The choice follows from the sizes alone; a thread keeps the last ones (the search takes 1 us).
Plan choose(const I8Product& p) {
    struct Kept { int M = 0, K = 0, N = 0, sms = 0; Plan plan; };
    static thread_local Kept kept[16];
    const int sms = num_sms();
    Kept& k = kept[(static_cast<unsigned>(p.M) * 31u + static_cast<unsigned>(p.K) * 7u + static_cast<unsigned>(p.N)) >> 3 & 15u];
    if (k.M != p.M || k.K != p.K || k.N != p.N || k.sms != sms) k = Kept{p.M, p.K, p.N, sms, choose_anew(p)};
    return k.plan;
}

template <typename T, int MORE>
int launch_t(const I8Product& p, const Plan& plan, cudaStream_t st) {
    const int cg = plan.pair == 2 ? 2 : 1;
    I8Tc q{};
    q.p = p; q.bn = plan.bn;
    q.stage_bytes = kABytes + plan.bn / cg * 128;
    q.stages = (kSmemMax - kBarBytes - kScaleBytes) / q.stage_bytes;
    if (q.stages > kMaxStages) q.stages = kMaxStages;
    q.kblocks = (p.K + 127) / 128;
    q.tiles_n = static_cast<int>((p.N + static_cast<long long>(kRowsA) * cg - 1) / (kRowsA * cg));
    q.tiles_t = static_cast<int>((p.M + static_cast<long long>(plan.bn) - 1) / plan.bn);
    if (static_cast<long long>(q.tiles_n) * q.tiles_t > INT32_MAX / 8) return ST_UNSUPPORTED_PATH;
    q.err = device_error_ptr();
    if (!q.err) return ST_LAUNCH;
    CUtensorMap tmW, tmA;
    if (!make_tmap_3d(&tmW, TmaType::U8, p.B, p.K, p.N, 1, p.ldb, 0, 128, kRowsA, 1) ||
        !make_tmap_3d(&tmA, TmaType::U8, p.A, p.K, p.M, 1, p.lda, 0, 128, plan.bn / cg, 1))
        return ST_UNSUPPORTED_PATH;
    const size_t smem = static_cast<size_t>(q.stages) * q.stage_bytes + kBarBytes + kScaleBytes;
    cudaError_t e;
    if (plan.pair == 0) {
        q.tmem_cols = pow2_at_least(plan.bn, 32);
        e = launch_cluster<i8_parts_kernel<T, MORE>>(q.tiles_n * q.tiles_t * plan.parts, plan.parts, smem, st, tmW, tmA, q, plan.parts);
    } else {
        q.tmem_cols = 2 * pow2_at_least(plan.bn, 32);
        const int units = q.tiles_n * q.tiles_t, most = num_sms() / cg, groups = units < most ? units : most;
        e = cg == 2 ? launch_cluster<i8_tiles_kernel<T, 2, MORE>>(groups * 2, 2, smem, st, tmW, tmA, q)
                    : launch_cluster<i8_tiles_kernel<T, 1, MORE>>(groups, 1, smem, st, tmW, tmA, q);
    }
    if (e != cudaSuccess) { cudaGetLastError(); return ST_LAUNCH; }
    return ST_OK;
}

template <typename T>
int launch_more(const I8Product& p, const Plan& plan, cudaStream_t st) {
    return p.gate ? launch_t<T, 2>(p, plan, st) : p.act ? launch_t<T, 1>(p, plan, st) : launch_t<T, 0>(p, plan, st);
}

}  // namespace

int launch_umma_i8(const I8Product& p, cudaStream_t st) {
    if (p.ldc > UINT32_MAX) return ST_UNSUPPORTED_PATH;
    if ((reinterpret_cast<uintptr_t>(p.A) | reinterpret_cast<uintptr_t>(p.B) | p.lda | p.ldb) & 15) return ST_UNSUPPORTED_PATH;
    const Plan plan = choose(p);
    switch (p.c_type) {
        case kTypeF32: return launch_more<float>(p, plan, st);
        case kTypeF16: return launch_more<__half>(p, plan, st);
        default: return launch_more<__nv_bfloat16>(p, plan, st);
    }
}

}  // namespace ppml_b200
