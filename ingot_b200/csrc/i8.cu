// W8A8 linear on int8 rows: Y[t, o] (+)= (sum_k X[t, k] W[o, k]) * sx[t] * sw[o], both sides int8 with a scale per row, weights packed once.
// The sums are exact integers (k up to 131,056), so that neither tiling nor a division of k changes a bit of the result.
//
//   D[128 features, BN tokens] += W[128, 128 bytes] * X[BN, 128 bytes]^T      per step of 128 inputs, tcgen05 kind::i8, s32 in tensor memory
#include <string.h>

#include <algorithm>

#include "internal.h"
#include "ptx.cuh"
#include "umma_i8.cuh"

namespace iq {

int32_t make_map_2d(iq_ctx* ctx, CUtensorMap* map, const void* base, int elem, uint64_t inner, uint64_t rows, uint64_t row_bytes, uint32_t box_inner,
                    uint32_t box_rows, bool swizzle128);

namespace {

constexpr int kI8MaxK = 131056;  // 131,056 * 128 * 128 < 2^31
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
    int32_t y_dtype, accumulate;
    int32_t M, N, K;
    int32_t m_tiles, steps;  // tiles of BN tokens; steps of 128 inputs
    int32_t* status;
};

template <int BN>
struct I8Tile {
    static constexpr int STAGE = 128 * 128 + BN * 128;
    static constexpr int PER_SM = BN <= 64 ? 2 : 1;
    static constexpr int FIT = (BN <= 64 ? 110 : 220) * 1024 / STAGE;
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
    static constexpr int SMEM = STAGES * STAGE + 1024 + 256;  // alignment, barriers
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

// A tile per cluster; its CTAs divide the steps among them and add their sums through distributed shared memory.
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
        if (__all_sync(0xffffffffu, mbar_wait(sums, 0, abort_flag))) {
            tc_fence_after();
            const int n = n0 + 32 * q + lane;
            const float sw = n < p.N ? p.sw[n] : 0.f;
            int* const park = reinterpret_cast<int*>(smem);  // [token][128 features]
            for (int c0 = 0; c0 < rows; c0 += 16) {
                uint32_t r[16];
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                             : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                               "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                             : "r"(t0 + c0)
                             : "memory");
                tmem_ld_wait();
                if (parts > 1) {
#pragma unroll
                    for (int j = 0; j < 16; j++) park[(c0 + j) * 128 + 32 * q + lane] = (int)r[j];
                } else if (n < p.N) {
#pragma unroll
                    for (int j = 0; j < 16; j++)
                        if (c0 + j < rows) {
                            const size_t o = (size_t)(row0 + c0 + j) * p.ldy + n;
                            float v = __fmul_rn(__fmul_rn((float)(int)r[j], p.sx[row0 + c0 + j]), sw);
                            if (p.accumulate) v += y_load(p.y, p.y_dtype, o);
                            y_store(p.y, p.y_dtype, o, v);
                        }
                }
            }
        }
    }
    __syncwarp();
    if (*abort_flag && warp == 0) {  // copies in flight land before the shared memory is given back
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {}
    }
    tc_fence_before();
    __syncthreads();
    if (parts > 1) {
        cluster_sync_all();  // every CTA's sums lie in its shared memory
        if (warp >= 2 && !*abort_flag) {
            // this CTA's share of the tile, four features at a time
            const int units = rows * 32, u0 = units * part / parts, u1 = units * (part + 1) / parts;
            for (int u = u0 + (int)threadIdx.x - 64; u < u1; u += 128) {
                int4 v = make_int4(0, 0, 0, 0);
                for (int c = 0; c < parts; c++) {
                    const int4 o = ld_dsmem_s4(smem_u32(smem) + u * 16, c);
                    v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
                }
                const int t = row0 + u / 32, n = n0 + u % 32 * 4;
                const float sx = p.sx[t];
                const int k[4] = {v.x, v.y, v.z, v.w};
                const size_t o = (size_t)t * p.ldy + n;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (n + j < p.N) {
                        float f = __fmul_rn(__fmul_rn((float)k[j], sx), p.sw[n + j]);
                        if (p.accumulate) f += y_load(p.y, p.y_dtype, o + j);
                        y_store(p.y, p.y_dtype, o + j, f);
                    }
            }
        }
        cluster_sync_all();  // nobody reads this CTA's shared memory any more
    }
    if (*abort_flag && threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, kErrTimeout);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(T::COLS) : "memory");
    }
}

typedef void (*I8Kernel)(CUtensorMap, CUtensorMap, I8Params);
struct I8Entry {
    int bn;
    void (*fn)(const CUtensorMap, const CUtensorMap, const I8Params);
    int smem, per_sm;
};
template <int BN>
constexpr I8Entry i8_entry() { return I8Entry{BN, i8_cluster_kernel<BN>, I8Tile<BN>::SMEM, I8Tile<BN>::PER_SM}; }
const I8Entry kI8[] = {i8_entry<16>(), i8_entry<32>(), i8_entry<64>(), i8_entry<128>(), i8_entry<256>()};

}  // namespace

int32_t i8_init(iq_ctx* ctx) {
    for (const I8Entry& e : kI8) {
        const cudaError_t r = cudaFuncSetAttribute(reinterpret_cast<const void*>(e.fn), cudaFuncAttributeMaxDynamicSharedMemorySize, e.smem);
        if (r != cudaSuccess) return check_cuda(ctx, r, "cudaFuncSetAttribute(i8)");
    }
    return kOk;
}

}  // namespace iq

using namespace iq;

extern "C" int32_t iq_qmm_i8(iq_ctx* ctx, void* stream, const int8_t* x, int64_t ldx, const float* x_scales, const int8_t* w, const float* w_scales,
                             int32_t n, int32_t k, void* y, int32_t y_dtype, int64_t ldy, int32_t rows, uint32_t flags) {
    // (the checks come before the context is looked at: they are the same without a GPU)
    if (x == nullptr || x_scales == nullptr || w == nullptr || w_scales == nullptr || y == nullptr || y_dtype < 0 || y_dtype > 2)
        return fail(ctx, kErrInvalidArg, "qmm_i8: null pointer, or y is not of fp32, fp16 or bf16");
    if (rows < 0 || n < 1 || k < 16 || k % 16 != 0) return fail(ctx, kErrInvalidArg, "qmm_i8: rows = %d, n = %d, k = %d (a multiple of 16)", rows, n, k);
    if (k > kI8MaxK) return fail(ctx, kErrUnsupported, "qmm_i8: k = %d (up to %d: sums in 32 bits)", k, kI8MaxK);
    if (ldx < k || ldx % 16 != 0 || ldy < n || reinterpret_cast<uintptr_t>(x) % 16 != 0 || reinterpret_cast<uintptr_t>(w) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(y) % dtype_size(y_dtype) != 0)
        return fail(ctx, kErrInvalidArg, "qmm_i8: x and w 16-byte aligned, ldx >= k a multiple of 16, ldy >= n");
    if ((flags & ~(uint32_t)IQ_FLAG_ACCUMULATE) != 0) return fail(ctx, kErrInvalidArg, "qmm_i8: flags %u", flags);
    if (ctx == nullptr) return kErrInvalidArg;
    if (rows == 0) return kOk;
    const I8Entry* e = kI8;
    while (e->bn < rows && e->bn < 256) e++;
    I8Params p;
    p.sx = x_scales; p.sw = w_scales; p.y = y; p.ldy = ldy; p.y_dtype = y_dtype; p.accumulate = flags & IQ_FLAG_ACCUMULATE ? 1 : 0;
    p.M = rows; p.N = n; p.K = k;
    p.m_tiles = (rows + e->bn - 1) / e->bn; p.steps = (k + 127) / 128; p.status = ctx->d_status;
    const int64_t tiles = (int64_t)p.m_tiles * ((n + 127) / 128);
    if (tiles > (1 << 27)) return fail(ctx, kErrUnsupported, "qmm_i8: %lld tiles", (long long)tiles);
    int parts = 1;
    while (parts < 8 && tiles * parts * 2 <= (int64_t)ctx->sms * e->per_sm && p.steps >= 4 * parts) parts *= 2;
    DeviceScope on(ctx);
    if (on.error != cudaSuccess) return check_cuda(ctx, on.error, "qmm_i8 device");
    CUtensorMap mx, mw;
    int32_t st = make_map_2d(ctx, &mx, x, 0, (uint64_t)k, (uint64_t)rows, (uint64_t)ldx, 128, (uint32_t)e->bn, true);
    if (st == kOk) st = cached_rows_map(ctx, w, n, k, 128, &mw);
    if (st != kOk) return st;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)(tiles * parts), 1, 1);
    cfg.blockDim = dim3(kI8Threads, 1, 1);
    cfg.dynamicSmemBytes = e->smem;
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return check_cuda(ctx, cudaLaunchKernelEx(&cfg, e->fn, mx, mw, p), "qmm_i8 launch");
}
