// W8A8 linear on int8 rows: Y[t, o] (+)= (sum_k X[t, k] W[o, k]) * sx[t] * sw[o], both sides int8 with a scale per row, weights packed once.
// The sums are exact integers (k up to 131,056), so that neither tiling nor a division of k changes a bit of the result.
//
//   D[128 features, BN tokens] += W[128, 128 bytes] * X[BN, 128 bytes]^T      per step of 128 inputs, tcgen05 kind::i8, s32 in tensor memory
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "ptx.cuh"
#include "umma_i8.cuh"

namespace iq {

int32_t make_map_2d(iq_ctx* ctx, CUtensorMap* map, const void* base, int elem, uint64_t inner, uint64_t rows, uint64_t row_bytes, uint32_t box_inner,
                    uint32_t box_rows, bool swizzle128);

namespace {

constexpr int kI8MaxK = 131056;  // 131,056 * 128 * 128 < 2^31
constexpr int kI8Most = 1 << 30;  // rows, features and CTAs
// kind::i8: s32 sums, signed 8-bit operands, both K-major, M = 128, N = n
__device__ __forceinline__ uint32_t i8_idesc(int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (8u << 24); }
// K-major rows of 128 bytes with the 128-byte swizzle
__device__ __forceinline__ uint64_t i8_desc(uint32_t saddr) { return kQtDescHi | (uint64_t)((saddr & 0x3FFFFu) >> 4); }

constexpr int kI8Threads = 192;  // copies, MMAs, four warps for the results

struct I8Params {
    const float* sx;
    const float* sw;
    void* y;
    int64_t ldy;
    int32_t y_dtype, accumulate, whole;  // whole: four neighbouring elements of y lie on their own size
    int32_t M, N;
    int32_t m_tiles, steps;  // tiles of tokens; steps of 128 inputs
    int32_t tile_rows, tall;  // pairs: tokens of the first `tall` of the tiles over the rows; the others have 32 fewer
    int32_t* status;
};

template <int BN>
struct I8Tile {
    static constexpr int STAGE = 128 * 128 + BN * 128;
    static constexpr int STAGES = 4;  // (two or three CTAs per SM; with three stages the next call starts earlier but 37 rows take 5 to 15 % longer)
    static constexpr int SMEM = STAGES * STAGE + 1024 + 256;  // alignment, barriers
    static constexpr int PER_SM = 227 * 1024 / (SMEM + 1024);
    static constexpr uint32_t COLS = BN < 32 ? 32 : BN;
    static_assert(BN * 512 <= STAGES * STAGE, "the partial sums take the stages' place");
};

__device__ __forceinline__ float y_load(const void* y, int32_t dtype, size_t i) {
    if (dtype == kF32) return static_cast<const float*>(y)[i];
    const uint16_t h = static_cast<const uint16_t*>(y)[i];
    return dtype == kBF16 ? bf16_bits_to_f32(h) : __half2float(__ushort_as_half(h));
}
__device__ __forceinline__ void y_store(void* y, int32_t dtype, size_t i, float v) {
    if (dtype == kF32) static_cast<float*>(y)[i] = v;
    else static_cast<uint16_t*>(y)[i] = dtype == kBF16 ? (uint16_t)f32_to_bf16_bits(v) : __half_as_ushort(__float2half_rn(v));
}
__device__ __forceinline__ int4 ld_dsmem_s4(uint32_t local, uint32_t cta) {
    int4 v;
    asm volatile("{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %4, %5;\nld.shared::cluster.v4.s32 {%0,%1,%2,%3}, [r];\n}\n"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(local), "r"(cta)
                 : "memory");
    return v;
}

// C neighbouring tokens of one feature: scaled, added, rounded and stored. sx: the scale of token `lane`; live: how many there are.
template <int DT, int C>
__device__ __forceinline__ void i8_store(const I8Params& p, const uint32_t (&r)[C], float sx, float sw, int row, int n, int live) {
    typedef typename std::conditional<DT == kF32, float, uint16_t>::type E;
    E* const y = static_cast<E*>(p.y) + (size_t)row * p.ldy + n;
    float v[C];
#pragma unroll
    for (int j = 0; j < C; j++) v[j] = __fmul_rn(__fmul_rn((float)(int)r[j], __shfl_sync(0xffffffffu, sx, j)), sw);
    if (n >= p.N) live = 0;
    if (p.accumulate) {  // all loads before the first store
#pragma unroll
        for (int j = 0; j < C; j++)
            if (j < live) v[j] += y_load(y, DT, (size_t)j * p.ldy);
    }
    if (live >= C) {
#pragma unroll
        for (int j = 0; j < C; j++) y_store(y, DT, (size_t)j * p.ldy, v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < C; j++)
            if (j < live) y_store(y, DT, (size_t)j * p.ldy, v[j]);
    }
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
// The lanes' features and C tokens of an accumulator to y
template <int C>
__device__ __forceinline__ void i8_results(const I8Params& p, uint32_t taddr, float sx, float sw, int row, int n, int live) {
    uint32_t r[C];
    tmem_ld(taddr, r);
    tmem_ld_wait();
    if (p.y_dtype == kF32) i8_store<kF32, C>(p, r, sx, sw, row, n, live);
    else if (p.y_dtype == kBF16) i8_store<kBF16, C>(p, r, sx, sw, row, n, live);
    else i8_store<kF16, C>(p, r, sx, sw, row, n, live);
}
// Sums of a token and four neighbouring features, the first of them n
template <int DT>
__device__ __forceinline__ void i8_store4(const I8Params& p, const int4& s, float sx, const float (&sw)[4], int row, int n) {
    typedef typename std::conditional<DT == kF32, float, uint16_t>::type E;
    E* const y = static_cast<E*>(p.y) + (size_t)row * p.ldy + n;
    const int k[4] = {s.x, s.y, s.z, s.w}, live = p.N - n;
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; j++) f[j] = __fmul_rn(__fmul_rn((float)k[j], sx), sw[j]);
    if (p.accumulate) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < live) f[j] += y_load(y, DT, j);
    }
    if (live >= 4 && p.whole) {
        if (DT == kF32) *reinterpret_cast<float4*>(y) = make_float4(f[0], f[1], f[2], f[3]);
        else if (DT == kF16) *reinterpret_cast<uint2*>(y) = make_uint2(pack_half2(f[0], f[1]), pack_half2(f[2], f[3]));
        else *reinterpret_cast<uint2*>(y) = make_uint2(f32_to_bf16_bits(f[0]) | f32_to_bf16_bits(f[1]) << 16, f32_to_bf16_bits(f[2]) | f32_to_bf16_bits(f[3]) << 16);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < live) y_store(y, DT, j, f[j]);
    }
}

// A thread's share of the results of 128 features from n0 on, in units of a token and four features (u0 + thread, and so on up to u1): the sums of PARTS CTAs of the
// cluster, which parked them at `park`, [token][128 features]. Eight loads of 16 bytes are under way at once. sx, sw: the scales of the first unit.
// Every load is waited for by a store of this thread ahead of the cluster's last meeting, which orders no memory: whoever owns it may leave after that.
// So a thread whose features lie beyond n loads nothing (of the last tile's odd CTAs, where n % 256 is 1 to 128, no thread does).
template <int PARTS, int THREADS, int STEP>
__device__ __forceinline__ void i8_shares(const I8Params& p, uint32_t park, uint32_t first, int u0, int u1, int row0, int n0, float sx0, const float (&sw)[4]) {
    static_assert(THREADS % 32 == 0, "a thread's units are of the same features");
    constexpr int B = 8 / PARTS;
    const int n = n0 + u0 % 32 * 4;
    if (n >= p.N) return;
    for (int u = u0; u < u1; u += B * THREADS) {
        int4 o[B][PARTS];
        float sx[B];
#pragma unroll
        for (int b = 0; b < B; b++)
            if (u + b * THREADS < u1) {
#pragma unroll
                for (int c = 0; c < PARTS; c++) o[b][c] = ld_dsmem_s4(park + (u + b * THREADS) * 16, first + STEP * c);
                sx[b] = u + b == u0 ? sx0 : p.sx[row0 + (u + b * THREADS) / 32];
            }
#pragma unroll
        for (int b = 0; b < B; b++) {
            if (u + b * THREADS >= u1) break;
            int4 v = o[b][0];
#pragma unroll
            for (int c = 1; c < PARTS; c++) { v.x += o[b][c].x; v.y += o[b][c].y; v.z += o[b][c].z; v.w += o[b][c].w; }
            const int t = row0 + (u + b * THREADS) / 32;
            if (p.y_dtype == kF32) i8_store4<kF32>(p, v, sx[b], sw, t, n);
            else if (p.y_dtype == kBF16) i8_store4<kBF16>(p, v, sx[b], sw, t, n);
            else i8_store4<kF16>(p, v, sx[b], sw, t, n);
        }
    }
}

// A tile per cluster; its CTAs divide the steps among them and add their sums through distributed shared memory.
//
// Bound: the weights' way from memory, and per call some 4 us of start (1 us from the kernel before to the first activations), sums of the cluster (2) and
// end. Four stages per CTA of the next call are loaded meanwhile. One row: 14336 x 4096 12.9 us (floor 9.0), 28672 x 4096 19.2 (18.0), 128,000 x 2048
// 40.7 (40.2). Asking for further weights into L2 ahead of the wait made it slower (12.9 -> 13.4 us with four more steps, 15.6 with all: the copies queue up
// before the activations'), and so did L2 promotion by 256 bytes (no effect) and tiles of 128 and 256 tokens (64 rows 8.7 us, 128 on one tile 11.1 and
// on two 9.2).
template <int BN>
__global__ void __launch_bounds__(kI8Threads, I8Tile<BN>::PER_SM)
    i8_cluster_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const I8Params p) {
    using T = I8Tile<BN>;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + T::STAGES * T::STAGE);  // full, empty, sums
    const uint32_t full = smem_u32(bars), empty = full + 8 * T::STAGES, sums = empty + 8 * T::STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * T::STAGES + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = gridDim.x / (p.m_tiles * ((p.N + 127) / 128)), part = (int)cluster_rank();
    const int tile = blockIdx.x / parts, row0 = (tile % p.m_tiles) * BN, n0 = (tile / p.m_tiles) * 128;
    const int rows = min(BN, p.M - row0);
    const int ks0 = p.steps * part / parts, ks1 = p.steps * (part + 1) / parts;
    if (threadIdx.x == 0) {
        for (int s = 0; s < T::STAGES; s++) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        mbar_init(sums, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(T::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    // a divided tile: this CTA's share of it, in units of a token and four features, and the scales of a thread's unit (the first: ahead of the sums)
    const int units = rows * 32, u0 = units * part / parts, u1 = units * (part + 1) / parts;
    float unit_sx = 0.f, unit_sw[4];
    auto unit_scales = [&](int u) {
        const int n = n0 + u % 32 * 4;
        unit_sx = p.sx[row0 + u / 32];
#pragma unroll
        for (int j = 0; j < 4; j++) unit_sw[j] = n + j < p.N ? p.sw[n + j] : 0.f;
    };
    if (warp == 0) {
        // ---- copies: the first stages' weights ahead of the wait for the kernel before (nothing of this library's that runs beside its
        // successor writes weights)
        if (elect_one()) {
            const int ahead = min(T::STAGES, ks1 - ks0);
            for (int s = 0; s < ahead; s++) {
                mbar_arrive_expect_tx(full + 8 * s, T::STAGE);
                tma_load_2d(smem_u32(smem + s * T::STAGE), &map_w, full + 8 * s, (ks0 + s) * 128, n0);
            }
            pdl_wait();
            for (int s = 0; s < ahead; s++) tma_load_2d(smem_u32(smem + s * T::STAGE) + 128 * 128, &map_x, full + 8 * s, (ks0 + s) * 128, row0);
            int s = 0;
            uint32_t ph = 0;
            for (int ks = ks0 + ahead; ks < ks1; ks++) {
                if (!mbar_wait(empty + 8 * s, ph, abort_flag)) break;
                const uint32_t st = smem_u32(smem + s * T::STAGE);
                mbar_arrive_expect_tx(full + 8 * s, T::STAGE);
                tma_load_2d(st, &map_w, full + 8 * s, ks * 128, n0);
                tma_load_2d(st + 128 * 128, &map_x, full + 8 * s, ks * 128, row0);
                if (++s == T::STAGES) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = i8_idesc((rows + 15) & ~15);
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int ks = ks0; ks < ks1; ks++) {
                if (!(ok = mbar_wait(full + 8 * s, ph, abort_flag))) break;
                tc_fence_after();
                const uint32_t st = smem_u32(smem + s * T::STAGE);
                const uint64_t a = i8_desc(st), b = i8_desc(st + 128 * 128);
#pragma unroll
                for (int kk = 0; kk < 4; kk++) umma_i8(tmem, a + 2 * kk, b + 2 * kk, idesc, (ks != ks0 || kk != 0) ? 1u : 0u);
                umma_commit(empty + 8 * s);
                if (++s == T::STAGES) { s = 0; ph ^= 1; }
            }
            if (ok) umma_commit(sums);
        }
    } else {
        pdl_wait();
        const int q = warp & 3;  // the quarter of tensor memory that this warp may read
        const uint32_t t0 = tmem + ((uint32_t)(32 * q) << 16);
        constexpr int C = 16;
        if (parts > 1 && u0 + (int)threadIdx.x < u1) unit_scales(u0 + (int)threadIdx.x);
        const int n = n0 + 32 * q + lane;
        const float sw = n < p.N ? p.sw[n] : 0.f, sx0 = lane < rows ? p.sx[row0 + lane] : 0.f, sx1 = 32 + lane < rows ? p.sx[row0 + 32 + lane] : 0.f;
        if (__all_sync(0xffffffffu, mbar_wait(sums, 0, abort_flag))) {
            tc_fence_after();
            int* const park = reinterpret_cast<int*>(smem);  // [token][128 features]
            for (int c0 = 0; c0 < rows; c0 += C) {
                if (parts == 1) {
                    i8_results<C>(p, t0 + c0, __shfl_sync(0xffffffffu, c0 < 32 ? sx0 : sx1, (lane + c0) & 31), sw, row0 + c0, n, rows - c0);
                } else {
                    uint32_t r[C];
                    tmem_ld(t0 + c0, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < C; j++) park[(c0 + j) * 128 + 32 * q + lane] = (int)r[j];
                }
            }
        }
    }
    __syncwarp();
    if (parts > 1 && warp < 2) {
        pdl_wait();
        if (u0 + (int)threadIdx.x < u1) unit_scales(u0 + (int)threadIdx.x);
    }
    if (*abort_flag && warp == 0) {  // copies in flight land before the shared memory is given back
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {}
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {  // (ahead of the cluster's meeting: a CTA that waits for others holds no tensor memory that theirs, or another kernel's, may be waiting for)
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(T::COLS) : "memory");
    }
    if (parts > 1) {
        cluster_sync_all();  // every CTA's sums lie in its shared memory
        if (!*abort_flag) {
            const uint32_t park = smem_u32(smem);
            const int u = u0 + (int)threadIdx.x;
            if (parts == 2) i8_shares<2, kI8Threads, 1>(p, park, 0, u, u1, row0, n0, unit_sx, unit_sw);
            else if (parts == 4) i8_shares<4, kI8Threads, 1>(p, park, 0, u, u1, row0, n0, unit_sx, unit_sw);
            else i8_shares<8, kI8Threads, 1>(p, park, 0, u, u1, row0, n0, unit_sx, unit_sw);
        }
        // nobody reads this CTA's shared memory any more (every load has gone into a sum that was stored: no ordering of memory to wait for)
        __syncwarp();
        asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    }
    if (*abort_flag && threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, kErrTimeout);
}

// ---- many rows: tiles of 256 features and up to 256 tokens on pairs of CTAs -----------------------------------------------
constexpr int kI8PairThreads = 320;  // copies, MMAs, eight warps for the results
constexpr int kI8PairStage = 2 * 128 * 128;  // of a CTA: its 128 features and its half of the tokens
constexpr int kI8PairStages = 6;
constexpr int kI8PairSmem = kI8PairStages * kI8PairStage + 1024 + 256;

__device__ __forceinline__ void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc)
        : "memory");
}
// Tensor copy into this CTA's shared memory whose bytes count on the barrier at this offset of the pair's even CTA, the cluster's CTA `even`
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, uint32_t even = 0) {
    asm volatile(
        "{\n.reg .b32 r;\nmapa.shared::cluster.u32 r, %2, %5;\n"
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [r];\n}\n"
        ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(even)
        : "memory");
}

// Persistent; two accumulators in tensor memory, so that a tile's results leave beside the next tile's products. The even CTA issues the
// MMAs for both; each copies its 128 features and its half of the tokens and stores its 128 features' results.
//
// Bound: operands on their way from L2 (a step of 128 inputs moves 16 KB + 64 bytes per token and SM, at some 46 bytes per cycle: 0.36 us on 256 tokens,
// the MMAs alone 0.27) and power. 2048 x 4096 x 14336 79 to 98 us, 2048 x 14336 x 4096 82, 4096 x 14336 x 4096 156 (3080 TOP/s). Measured and taken
// back: 512 tokens per pair as two MMAs on the same features (the step 11 % shorter per token, but no room for a second accumulator: 84 us against 79).
// Stages of 96 KB, so that the next call's CTAs start beside this one's: they gather on the same SMs (256 x 4096 x 14336 20.1 -> 25.8 us).
__global__ void __launch_bounds__(kI8PairThreads, 1) __cluster_dims__(2, 1, 1)
    i8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const I8Params p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kI8PairStages * kI8PairStage);  // full, empty; accumulators full [2], empty [2]
    const uint32_t full = smem_u32(bars), empty = full + 8 * kI8PairStages, tfull = empty + 8 * kI8PairStages, tempty = tfull + 16;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kI8PairStages + 4);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kI8PairStages; s++) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(tfull + 8 * a, 1);
            mbar_init(tempty + 8 * a, 16);  // both CTAs' eight warps
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // the other CTA's barriers exist
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    const int total = p.m_tiles * ((p.N + 255) / 256), first = blockIdx.x / 2, stride = gridDim.x / 2;
    const uint32_t bytes = 128 * 128 + p.tile_rows * 64;  // of a CTA and stage
    // tile m over the rows: its first row, its rows, and the tokens of its MMAs: whole groups of 32, half of them in each CTA
    auto first_row = [&](int m) { return m * p.tile_rows - 32 * max(m - p.tall, 0); };
    auto tile_rows = [&](int m) { return min(p.tile_rows - (m < p.tall ? 0 : 32), p.M - first_row(m)); };
    auto tokens = [&](int m) { return (tile_rows(m) + 31) & ~31; };
    if (warp == 0) {
        if (elect_one()) {
            auto corner = [&](int i, int& xrow, int& n0) {
                const int m = i % p.m_tiles;
                n0 = (i / p.m_tiles) * 256 + 128 * (int)rank;
                xrow = first_row(m) + (int)rank * (tokens(m) / 2);
            };
            // the first stages' weights ahead of the wait for the kernel before
            int xrow, n0;
            corner(first, xrow, n0);
            const int ahead = min(kI8PairStages, p.steps);
            for (int s = 0; s < ahead; s++) {
                if (rank == 0) mbar_arrive_expect_tx(full + 8 * s, 2 * bytes);
                tma_load_2d_pair(smem_u32(smem + s * kI8PairStage), &map_w, full + 8 * s, s * 128, n0);
            }
            pdl_wait();
            for (int s = 0; s < ahead; s++) tma_load_2d_pair(smem_u32(smem + s * kI8PairStage) + 128 * 128, &map_x, full + 8 * s, s * 128, xrow);
            int s = ahead % kI8PairStages;
            uint32_t ph = ahead / kI8PairStages;
            bool ok = true;
            for (int i = first, ks = ahead; i < total && ok; i += stride, ks = 0) {
                corner(i, xrow, n0);
                for (; ks < p.steps; ks++) {
                    if (!(ok = mbar_wait(empty + 8 * s, ph ^ 1, abort_flag))) break;
                    const uint32_t st = smem_u32(smem + s * kI8PairStage);
                    if (rank == 0) mbar_arrive_expect_tx(full + 8 * s, 2 * bytes);
                    tma_load_2d_pair(st, &map_w, full + 8 * s, ks * 128, n0);
                    tma_load_2d_pair(st + 128 * 128, &map_x, full + 8 * s, ks * 128, xrow);
                    if (++s == kI8PairStages) { s = 0; ph ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            int s = 0, a = 0;
            uint32_t ph = 0, tph = 0;
            bool ok = true;
            for (int i = first; i < total && ok; i += stride) {
                const uint32_t idesc = i8_idesc(tokens(i % p.m_tiles)) + (8u << 24);  // M = 256
                if (!(ok = mbar_wait(tempty + 8 * a, tph ^ 1, abort_flag))) break;
                tc_fence_after();
                const uint32_t acc = tmem + a * 256;
                for (int ks = 0; ks < p.steps; ks++) {
                    if (!(ok = mbar_wait(full + 8 * s, ph, abort_flag))) break;
                    tc_fence_after();
                    const uint32_t st = smem_u32(smem + s * kI8PairStage);
                    const uint64_t ad = i8_desc(st), bd = i8_desc(st + 128 * 128);
#pragma unroll
                    for (int kk = 0; kk < 4; kk++) umma_i8_pair(acc, ad + 2 * kk, bd + 2 * kk, idesc, (ks | kk) != 0 ? 1u : 0u);
                    umma_commit_pair(empty + 8 * s);
                    if (++s == kI8PairStages) { s = 0; ph ^= 1; }
                }
                if (ok) umma_commit_pair(tfull + 8 * a);
                a ^= 1;
                if (a == 0) tph ^= 1;
            }
        }
    } else {
        pdl_wait();
        // Two times four warps take sixteen tokens in turn. (Thirty-two at once spill: 2048 x 4096 x 4096 30.7 us against 27.7, 2048 x 1024 x 1024 8.8 against 7.1.)
        constexpr int C = 16;
        const int q = warp & 3, half = (warp - 2) >> 2;
        int a = 0;
        uint32_t tph = 0;
        for (int i = first; i < total; i += stride) {
            const int row0 = first_row(i % p.m_tiles) + C * half, rows = tile_rows(i % p.m_tiles) - C * half;  // from the warp's first token on
            const int n = (i / p.m_tiles) * 256 + 128 * (int)rank + 32 * q + lane;
            const float sw = n < p.N ? p.sw[n] : 0.f;
            auto scale = [&](int c0) { return lane < C && c0 + lane < rows ? p.sx[row0 + c0 + lane] : 0.f; };
            float sx = scale(0);
            if (!__all_sync(0xffffffffu, mbar_wait(tfull + 8 * a, tph, abort_flag))) break;
            tc_fence_after();
            const uint32_t t0 = tmem + ((uint32_t)(32 * q) << 16) + a * 256 + C * half;
            uint32_t r[2][C];  // the next columns are under way while these are stored
            if (rows > 0) tmem_ld(t0, r[0]);
#pragma unroll 1
            for (int c2 = 0; c2 < rows; c2 += 4 * C) {
#pragma unroll
                for (int c1 = 0; c1 < 2; c1++) {
                    const int c0 = c2 + 2 * C * c1;
                    if (c0 >= rows) break;
                    const float next = scale(c0 + 2 * C);
                    tmem_ld_wait();
                    if (c0 + 2 * C < rows) tmem_ld(t0 + c0 + 2 * C, r[c1 ^ 1]);
                    if (p.y_dtype == kF32) i8_store<kF32, C>(p, r[c1], sx, sw, row0 + c0, n, rows - c0);
                    else if (p.y_dtype == kBF16) i8_store<kBF16, C>(p, r[c1], sx, sw, row0 + c0, n, rows - c0);
                    else i8_store<kF16, C>(p, r[c1], sx, sw, row0 + c0, n, rows - c0);
                    sx = next;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (rank != 0) mbar_arrive_remote(tempty + 8 * a, 0);
                else mbar_arrive(tempty + 8 * a);
            }
            a ^= 1;
            if (a == 0) tph ^= 1;
        }
    }
    __syncwarp();
    if (*abort_flag && warp == 0) {  // copies in flight land before the shared memory is given back
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {}
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // (the other CTA's MMAs read this one's memory, its arrivals go to this one's barriers)
    if (*abort_flag && threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, kErrTimeout);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Completion of all tcgen05.mma issued so far, to the barrier at this offset in both CTAs of the pair whose even one is the cluster's CTA `even`
__device__ __forceinline__ void umma_commit_pair_at(uint32_t bar, uint32_t even) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)(3u << even))
                 : "memory");
}

// Few tiles and many inputs: SPLIT pairs in a cluster divide a tile's steps, a tile per cluster. Every CTA parks its sums (its 128 features, int32) where its
// stages were, and finishes its share of the tokens from its SPLIT counterparts' memory.
template <int SPLIT>
__global__ void __launch_bounds__(kI8PairThreads, 1) __cluster_dims__(2 * SPLIT, 1, 1)
    i8_split_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const I8Params p) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kI8PairStages * kI8PairStage);  // full, empty, sums
    const uint32_t full = smem_u32(bars), empty = full + 8 * kI8PairStages, sums = empty + 8 * kI8PairStages;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kI8PairStages + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    static_assert(256 * 512 <= kI8PairStages * kI8PairStage, "the partial sums take the stages' place");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), half = rank & 1, even = rank & ~1u;
    const int part = (int)rank / 2, tile = blockIdx.x / (2 * SPLIT), m = tile % p.m_tiles;
    const int row0 = m * p.tile_rows - 32 * max(m - p.tall, 0), rows = min(p.tile_rows - (m < p.tall ? 0 : 32), p.M - row0), tokens = (rows + 31) & ~31;
    const int n0 = (tile / p.m_tiles) * 256 + 128 * (int)half;
    const int ks0 = p.steps * part / SPLIT, ks1 = p.steps * (part + 1) / SPLIT;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kI8PairStages; s++) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        mbar_init(sums, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(256) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // the other CTAs' barriers exist
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    const uint32_t bytes = 128 * 128 + p.tile_rows * 64;  // of a CTA and stage
    // this CTA's share of its features' results, in units of a token and four features, and the scales of a thread's unit (the first: ahead of the sums)
    const int units = rows * 32, u0 = units * part / SPLIT, u1 = units * (part + 1) / SPLIT;
    float unit_sx = 0.f, unit_sw[4];
    auto unit_scales = [&](int u) {
        const int n = n0 + u % 32 * 4;
        unit_sx = p.sx[row0 + u / 32];
#pragma unroll
        for (int j = 0; j < 4; j++) unit_sw[j] = n + j < p.N ? p.sw[n + j] : 0.f;
    };
    if (warp == 0) {
        if (elect_one()) {
            const int xrow = row0 + (int)half * (tokens / 2), ahead = min(kI8PairStages, ks1 - ks0);
            // the first stages' weights ahead of the wait for the kernel before
            for (int s = 0; s < ahead; s++) {
                if (half == 0) mbar_arrive_expect_tx(full + 8 * s, 2 * bytes);
                tma_load_2d_pair(smem_u32(smem + s * kI8PairStage), &map_w, full + 8 * s, (ks0 + s) * 128, n0, even);
            }
            pdl_wait();
            for (int s = 0; s < ahead; s++) tma_load_2d_pair(smem_u32(smem + s * kI8PairStage) + 128 * 128, &map_x, full + 8 * s, (ks0 + s) * 128, xrow, even);
            int s = ahead % kI8PairStages;
            uint32_t ph = 0;
            for (int ks = ks0 + ahead; ks < ks1; ks++) {
                if (!mbar_wait(empty + 8 * s, ph, abort_flag)) break;
                const uint32_t st = smem_u32(smem + s * kI8PairStage);
                if (half == 0) mbar_arrive_expect_tx(full + 8 * s, 2 * bytes);
                tma_load_2d_pair(st, &map_w, full + 8 * s, ks * 128, n0, even);
                tma_load_2d_pair(st + 128 * 128, &map_x, full + 8 * s, ks * 128, xrow, even);
                if (++s == kI8PairStages) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (half == 0 && elect_one()) {
            const uint32_t idesc = i8_idesc(tokens) + (8u << 24);  // M = 256
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int ks = ks0; ks < ks1; ks++) {
                if (!(ok = mbar_wait(full + 8 * s, ph, abort_flag))) break;
                tc_fence_after();
                const uint32_t st = smem_u32(smem + s * kI8PairStage);
                const uint64_t ad = i8_desc(st), bd = i8_desc(st + 128 * 128);
#pragma unroll
                for (int kk = 0; kk < 4; kk++) umma_i8_pair(tmem, ad + 2 * kk, bd + 2 * kk, idesc, (ks != ks0 || kk != 0) ? 1u : 0u);
                umma_commit_pair_at(empty + 8 * s, even);
                if (++s == kI8PairStages) { s = 0; ph ^= 1; }
            }
            if (ok) umma_commit_pair_at(sums, even);
        }
    } else {
        // two times four warps park sixteen tokens in turn
        constexpr int C = 16;
        const int q = warp & 3;
        int* const park = reinterpret_cast<int*>(smem) + 32 * q + lane;  // [token][128 features]
        if (__all_sync(0xffffffffu, mbar_wait(sums, 0, abort_flag))) {
            tc_fence_after();
            const uint32_t t0 = tmem + ((uint32_t)(32 * q) << 16);
            for (int c0 = C * ((warp - 2) >> 2); c0 < rows; c0 += 2 * C) {
                uint32_t r[C];
                tmem_ld(t0 + c0, r);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < C; j++) park[(c0 + j) * 128] = (int)r[j];
            }
        }
    }
    __syncwarp();
    pdl_wait();
    if (u0 + (int)threadIdx.x < u1) unit_scales(u0 + (int)threadIdx.x);
    if (*abort_flag && warp == 0) {  // copies in flight land before the shared memory is given back
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {}
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();  // every CTA's sums lie in its shared memory
    if (!*abort_flag) i8_shares<SPLIT, kI8PairThreads, 2>(p, smem_u32(smem), half, u0 + (int)threadIdx.x, u1, row0, n0, unit_sx, unit_sw);
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");  // (nobody reads this CTA's shared memory any more: i8_shares)
    if (*abort_flag && threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, kErrTimeout);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256) : "memory");
    }
}

struct I8Entry {
    int bn;
    void (*fn)(const CUtensorMap, const CUtensorMap, const I8Params);
    int smem;
};
template <int BN>
constexpr I8Entry i8_entry() { return I8Entry{BN, i8_cluster_kernel<BN>, I8Tile<BN>::SMEM}; }
const I8Entry kI8[] = {i8_entry<16>(), i8_entry<32>(), i8_entry<64>()};

// How a call is divided. Up to 128 rows clusters, which hide the weights' way from memory; beyond the cheapest by estimates in ns. A step on h tokens per
// tile takes a pair 180 + 0.5 h (and 0.6 more for each beyond 128), one of the pairs that divide a tile's steps 150 + 30 s + 0.4 h, a cluster's CTA on 64 tokens (two per
// SM) 330; start and end 4000 + 8 h, 3000 + 23 h (all of a tile's sums pass through shared memory), 5000 (one CTA alone 3700). Measured / estimated, us:
//                        clusters       pairs          two pairs      three pairs
//   256 x 4096 x 4096     10.6 / 10.3    11.0 / 11.3    10.2 / 10.2    12.1 / 12.3
//   512 x 4096 x 4096     13.2 / 14.3    13.0 / 12.9    13.9 / 13.9
//   256 x 4096 x 14336    23.2 / 23.5    26.9 / 28.3    20.1 / 20.6    21.0 / 21.9
//   512 x 4096 x 14336    37.1 / 40.7    30.2 / 32.4    26.3 / 26.4
//   160 x 4096 x 14336    22.9 / 23.5    26.7 / 27.9    18.7 / 18.4    17.9 / 18.3
//   3186 x 256 x 12928    21.7 / 21.8    24.9 / 25.9    17.6 / 18.0    16.2 / 16.5
// Four pairs were no better than three anywhere (15 clusters of eight CTAs run at once: 3186 x 256 x 12928 16.1, 703 x 1136 x 9216 13.9 against 13.0).
// The pairs' tiles over the rows are of two heights, 32 apart, so that any number of them can be had: sixteen times nine fill 74 pairs twice, sixteen times eight
// (of 256 tokens) did so to 86 %.
struct I8Plan {
    bool pair;
    int rows, tall;  // tokens of a tile; pairs: of the first `tall` over the rows, the others have 32 fewer
    int m_tiles;
    int64_t tiles;
    int parts;  // pieces of k: the CTAs of a cluster, or its pairs
};
// Clusters of so many CTAs that run at once, where an SM holds so many: each stays in one group of SMs. (Measured on 148 SMs: of four CTAs 33, 71 and 104 with one, two
// and three per SM, of six 22, of eight 33 and 48.)
int i8_at_once(int ctas, int per_sm, int sms) { return sms * 11 / 12 / ctas * per_sm; }
I8Plan i8_plan(int rows, int n, int k, int sms) {
    const int64_t steps = (k + 127) / 128;
    I8Plan c;
    c.pair = false;
    c.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    c.m_tiles = (rows + c.rows - 1) / c.rows;
    c.tall = c.m_tiles;
    c.tiles = (int64_t)c.m_tiles * ((n + 127) / 128);
    c.parts = 1;
    // (a division costs about 1 us: 37 x 1024 x 1024, eight steps, 4.2 us whole and 4.8 in four; 23 steps of 37 x 2880 x 2880 8.4 and 6.4. Clusters that do not
    // run at once: 64 x 4736 x 4096, 37 tiles, 8.7 us in four parts and 12.5 in eight, 64 x 9216 x 4096, 72 tiles, 12.1 in two and 15.8 in four)
    while (steps > 8 && c.parts < 8 && c.tiles * c.parts <= sms && steps >= 4 * c.parts && (c.parts == 1 || c.tiles <= i8_at_once(2 * c.parts, c.rows == 16 ? 3 : 2, sms)))
        c.parts *= 2;
    if (rows <= 128 || sms % 2 != 0 || c.tiles > kI8Most) return c;
    int64_t least = (c.tiles * c.parts + 2 * sms - 1) / (2 * sms) * (steps / c.parts) * 330 + (c.parts > 1 ? 5000 : 3700);
    const int n_tiles = (n + 255) / 256, groups = (rows + 31) / 32;
    for (int m = (groups + 7) / 8; m <= (groups + 1) / 2; m++) {
        const int high = (groups + m - 1) / m;  // groups of 32 tokens
        const int64_t tiles = (int64_t)m * n_tiles, rounds = (tiles + sms / 2 - 1) / (sms / 2), h = rows / m;
        const int64_t whole = rounds * steps * (1800 + 5 * h + 6 * std::max<int64_t>(h - 128, 0)) / 10 + 4000 + 8 * h;
        auto take = [&](int64_t cost, int parts) {
            if (cost >= least) return;
            least = cost;
            c = I8Plan{true, 32 * high, groups - m * (high - 1), m, tiles, parts};
        };
        take(whole, 1);
        for (int s = 2; s <= 3; s++)
            if (steps >= 4 * s && tiles <= i8_at_once(2 * s, 1, sms)) take((steps + s - 1) / s * (1500 + 300 * s + 4 * h) / 10 + 3000 + 23 * h, s);
        if (rounds > 64) break;  // (finer tiles only cost)
    }
    return c;
}

}  // namespace

int32_t i8_init(iq_ctx* ctx) {
    for (const I8Entry& e : kI8) {
        const cudaError_t r = cudaFuncSetAttribute(reinterpret_cast<const void*>(e.fn), cudaFuncAttributeMaxDynamicSharedMemorySize, e.smem);
        if (r != cudaSuccess) return check_cuda(ctx, r, "cudaFuncSetAttribute(i8)");
    }
    for (auto kernel : {i8_pair_kernel, i8_split_kernel<2>, i8_split_kernel<3>}) {
        const cudaError_t r = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, kI8PairSmem);
        if (r != cudaSuccess) return check_cuda(ctx, r, "cudaFuncSetAttribute(i8_pair)");
    }
    return kOk;
}

}  // namespace iq

using namespace iq;

extern "C" int32_t iq_qmm_i8_plan(int32_t rows, int32_t n, int32_t k, int32_t sms, iq_qmm_i8_tiling* out) {
    if (out == nullptr || rows < 1 || n < 1 || k < 16 || k % 16 != 0 || k > kI8MaxK || sms < 1) return kErrInvalidArg;
    if (rows > kI8Most || n > kI8Most) return kErrUnsupported;
    const I8Plan p = i8_plan(rows, n, k, sms);
    out->tile_rows = p.rows;
    out->tall = p.tall;
    out->row_tiles = p.m_tiles;
    out->pair = p.pair ? 1 : 0;
    out->parts = p.parts;
    out->tiles = p.tiles;
    return kOk;
}

extern "C" int32_t iq_qmm_i8(iq_ctx* ctx, void* stream, const int8_t* x, int64_t ldx, const float* x_scales, const int8_t* w, const float* w_scales,
                             int32_t n, int32_t k, void* y, int32_t y_dtype, int64_t ldy, int32_t rows, uint32_t flags) {
    // (the checks come before the context is looked at: they are the same without a GPU)
    if (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr || y == nullptr || y_dtype < 0 || y_dtype > 2)
        return fail(ctx, kErrInvalidArg, "qmm_i8: null pointer, or y is not of fp32, fp16 or bf16");
    if (rows < 0 || n < 1 || k < 16 || k % 16 != 0) return fail(ctx, kErrInvalidArg, "qmm_i8: rows = %d, n = %d, k = %d (a multiple of 16)", rows, n, k);
    if (k > kI8MaxK) return fail(ctx, kErrUnsupported, "qmm_i8: k = %d (up to %d: sums in 32 bits)", k, kI8MaxK);
    if (ldx < k || ldx % 16 != 0 || ldy < n || reinterpret_cast<uintptr_t>(x) % 16 != 0 || reinterpret_cast<uintptr_t>(w) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(y) % dtype_size(y_dtype) != 0 || (reinterpret_cast<uintptr_t>(x_scales) | reinterpret_cast<uintptr_t>(w_scales)) % 4 != 0)
        return fail(ctx, kErrInvalidArg, "qmm_i8: x and w 16-byte aligned, y and scales on their elements, ldx >= k a multiple of 16, ldy >= n");
    if (rows > kI8Most || n > kI8Most) return fail(ctx, kErrUnsupported, "qmm_i8: rows = %d, n = %d (up to %d)", rows, n, kI8Most);
    if ((flags & ~(uint32_t)IQ_FLAG_ACCUMULATE) != 0) return fail(ctx, kErrInvalidArg, "qmm_i8: flags %u", flags);
    if (ctx == nullptr) return kErrInvalidArg;
    if (rows == 0) return kOk;
    const I8Plan plan = i8_plan(rows, n, k, ctx->sms);
    if (plan.tiles * plan.parts > kI8Most) return fail(ctx, kErrUnsupported, "qmm_i8: %lld tiles", (long long)plan.tiles);
    I8Params p;
    p.sx = x_scales; p.sw = w_scales; p.y = y; p.ldy = ldy; p.y_dtype = y_dtype;
    p.accumulate = flags & IQ_FLAG_ACCUMULATE ? 1 : 0;
    p.whole = ldy % 4 == 0 && reinterpret_cast<uintptr_t>(y) % (4 * dtype_size(y_dtype)) == 0;
    p.M = rows; p.N = n;
    p.tile_rows = plan.rows; p.tall = plan.tall; p.m_tiles = plan.m_tiles; p.steps = (k + 127) / 128;
    p.status = ctx->d_status;
    DeviceScope on(ctx);
    if (on.error != cudaSuccess) return check_cuda(ctx, on.error, "qmm_i8 device");
    CUtensorMap mx, mw;
    int32_t st = make_map_2d(ctx, &mx, x, 0, (uint64_t)k, (uint64_t)rows, (uint64_t)ldx, 128, (uint32_t)(plan.pair ? plan.rows / 2 : plan.rows), true);
    if (st == kOk) st = make_map_2d(ctx, &mw, w, 0, (uint64_t)k, (uint64_t)n, (uint64_t)k, 128, 128, true);
    if (st != kOk) return st;
    cudaStream_t cs = reinterpret_cast<cudaStream_t>(stream);
    if (plan.pair && plan.parts > 1)
        return check_cuda(ctx, launch_dependent(plan.parts == 2 ? i8_split_kernel<2> : i8_split_kernel<3>, dim3((unsigned)(plan.tiles * plan.parts * 2)), kI8PairThreads,
                                                kI8PairSmem, cs, mx, mw, p),
                          "qmm_i8 launch");
    if (plan.pair)
        return check_cuda(ctx, launch_dependent(i8_pair_kernel, dim3((unsigned)std::min<int64_t>(plan.tiles, ctx->sms / 2) * 2), kI8PairThreads, kI8PairSmem, cs, mx, mw, p),
                          "qmm_i8 launch");
    const I8Entry* e = kI8;
    while (e->bn != plan.rows) e++;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)(plan.tiles * plan.parts), 1, 1);
    cfg.blockDim = dim3(kI8Threads, 1, 1);
    cfg.dynamicSmemBytes = e->smem;
    cfg.stream = cs;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = plan.parts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return check_cuda(ctx, cudaLaunchKernelEx(&cfg, e->fn, mx, mw, p), "qmm_i8 launch");
}
