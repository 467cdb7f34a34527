// The step between two sublayers: the residual's addition, the weighted RMS norm of the sum, and where the linears behind it are
// W8A8, its int8 codes with a scale per row, rotated as their weights are. One pass: a row stays in the registers of its block.
//
//   r' = round(r + x)                        x's rows may be absent (a stack's first norm): r' = r
//   q  = 1 / sqrt(mean(r'^2) + eps)
//   out = round((r' * q) * (w + offset))
//   v  = r' * (w + offset), u = H_n v        n = 1 (none), 32 or 256: per block of n inputs, spans 1, 2, 4, ...: a + b and a - b
//   s  = max|u| / 127, codes = rint(u / s) within -127..127, scale = s * q
//
// q is the same for a whole row, so the codes do not need it: every operation on their way is one fp32 operation on stored
// values, and the codes are the same bits whatever the launch looks like (only q's sum has an order). The steps from u on are those of
// the W8A8 GEMM's own conversion (w8a8.cu).
#include <cuda_bf16.h>

#include "common.cuh"
#include "internal.h"
#include "ptx.cuh"

namespace iq {
namespace {

constexpr int kNormMaxD = 32768;

struct NormParams {
    const void* x;
    const void* r;
    void* r_out;
    const void* w;
    void* out;
    int8_t* codes;
    float* scales;
    int64_t ldx, ldr, ldro, ldo, ldc;
    int32_t x_dtype, r_dtype, w_dtype, out_dtype;
    int32_t d;
    float offset, eps;
};

// Eight values as they lie in memory, and as floats. dtype is the same for a whole launch: a branch costs an issue slot.
struct Raw8 {
    uint4 a, b;
};
__device__ __forceinline__ Raw8 raw8_load(const void* p, int32_t dtype, size_t i) {
    Raw8 r;
    r.b = make_uint4(0, 0, 0, 0);
    if (dtype == kF32) {
        const uint4* q = reinterpret_cast<const uint4*>(static_cast<const float*>(p) + i);
        r.a = q[0];
        r.b = q[1];
    } else {
        r.a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    }
    return r;
}
__device__ __forceinline__ float scalar_load(const void* p, int32_t dtype, size_t i) {
    if (dtype == kF32) return static_cast<const float*>(p)[i];
    const uint16_t h = static_cast<const uint16_t*>(p)[i];
    return dtype == kBF16 ? bf16_bits_to_f32(h) : __half2float(__ushort_as_half(h));
}
__device__ __forceinline__ float round_to(float v, int32_t dtype) {
    if (dtype == kF32) return v;
    return dtype == kBF16 ? __bfloat162float(__float2bfloat16_rn(v)) : __half2float(__float2half_rn(v));
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, int32_t dtype) {
    if (dtype == kF16) return pack_half2(lo, hi);
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ void store8(void* p, int32_t dtype, size_t i, const float (&v)[8]) {
    if (dtype == kF32) {
        float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
        q[0] = make_float4(v[0], v[1], v[2], v[3]);
        q[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
            make_uint4(pack2(v[0], v[1], dtype), pack2(v[2], v[3], dtype), pack2(v[4], v[5], dtype), pack2(v[6], v[7], dtype));
    }
}
__device__ __forceinline__ void scalar_store(void* p, int32_t dtype, size_t i, float v) {
    if (dtype == kF32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = dtype == kBF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// A row per block, NCH times eight values per thread.
// VEC: rows of whole, 16-byte aligned groups of eight (codes: 8-byte aligned). Else value by value: neighbouring threads take
// neighbouring values, except where the rotation wants a thread to have eight in a row.
// CODES, ROT: int8 codes, rotated in blocks of ROT inputs (1: not): spans 1, 2, 4 inside a thread, the others between lanes.
template <int NCH, bool VEC, bool CODES, int ROT>
__global__ void __launch_bounds__(1024) add_rmsnorm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float wsum[32];
    __shared__ uint32_t wmax[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const size_t row = blockIdx.x;
    pdl_launch_dependents();
    constexpr bool RUNS = VEC || ROT > 1;  // a thread's eight values lie in a row
    auto at = [&](int c, int j) { return RUNS ? (c * (int)blockDim.x + tid) * 8 + j : (c * 8 + j) * (int)blockDim.x + tid; };
    pdl_wait();
    float v[NCH][8];  // r'
    if (VEC) {
        Raw8 rr[NCH], xx[NCH];
#pragma unroll
        for (int c = 0; c < NCH; c++)
            if (at(c, 0) < p.d) {
                rr[c] = raw8_load(p.r, p.r_dtype, row * p.ldr + at(c, 0));
                if (p.x != nullptr) xx[c] = raw8_load(p.x, p.x_dtype, row * p.ldx + at(c, 0));
            }
#pragma unroll
        for (int c = 0; c < NCH; c++) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[c][j] = 0.f;
            if (at(c, 0) < p.d) {
                unpack_x8(RawX8{rr[c].a, rr[c].b}, p.r_dtype, v[c]);
                if (p.x != nullptr) {
                    float xv[8];
                    unpack_x8(RawX8{xx[c].a, xx[c].b}, p.x_dtype, xv);
#pragma unroll
                    for (int j = 0; j < 8; j++) v[c][j] = round_to(v[c][j] + xv[j], p.r_dtype);
                    store8(p.r_out, p.r_dtype, row * p.ldro + at(c, 0), v[c]);
                }
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < NCH; c++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[c][j] = 0.f;
                if (at(c, j) < p.d) {
                    v[c][j] = scalar_load(p.r, p.r_dtype, row * p.ldr + at(c, j));
                    if (p.x != nullptr) v[c][j] = round_to(v[c][j] + scalar_load(p.x, p.x_dtype, row * p.ldx + at(c, j)), p.r_dtype);
                }
            }
        if (p.x != nullptr) {  // (behind all loads: r_out may be r)
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (at(c, j) < p.d) scalar_store(p.r_out, p.r_dtype, row * p.ldro + at(c, j), v[c][j]);
        }
    }
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) sum = fmaf(v[c][j], v[c][j], sum);
    // w + offset of the thread's values
    auto weights = [&](int c, float (&w)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = 1.f;
        if (p.w == nullptr) return;
        if (VEC) {
            if (at(c, 0) < p.d) {
                const Raw8 r = raw8_load(p.w, p.w_dtype, at(c, 0));
                unpack_x8(RawX8{r.a, r.b}, p.w_dtype, w);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (at(c, j) < p.d) w[j] = scalar_load(p.w, p.w_dtype, at(c, j));
        }
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = __fadd_rn(w[j], p.offset);
    };
    float u[CODES ? NCH : 1][8];
    uint32_t most = 0;  // largest |u| as bits: NaN and infinity are above every number
    if (CODES) {
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            float w[8];
            weights(c, w);
#pragma unroll
            for (int j = 0; j < 8; j++) u[c][j] = __fmul_rn(v[c][j], w[j]);
            if (ROT > 1) {
#pragma unroll
                for (int h = 1; h < 8; h <<= 1)
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if ((j & h) == 0) {
                            const float a = u[c][j], b = u[c][j + h];
                            u[c][j] = __fadd_rn(a, b);
                            u[c][j + h] = __fsub_rn(a, b);
                        }
#pragma unroll
                for (int h = 1; h < ROT / 8; h <<= 1)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float o = __shfl_xor_sync(0xffffffffu, u[c][j], h);
                        u[c][j] = (lane & h) ? __fsub_rn(o, u[c][j]) : __fadd_rn(u[c][j], o);
                    }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) most = max(most, __float_as_uint(u[c][j]) & 0x7FFFFFFFu);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) wmax[warp] = most;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) wsum[warp] = sum;
    __syncthreads();
    sum = lane < warps ? wsum[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float q = rsqrtf(__fadd_rn(__fdiv_rn(sum, (float)p.d), p.eps));
    if (p.out != nullptr) {
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            float w[8], o[8];
            weights(c, w);
#pragma unroll
            for (int j = 0; j < 8; j++) o[j] = (v[c][j] * q) * w[j];
            if (VEC) {
                if (at(c, 0) < p.d) store8(p.out, p.out_dtype, row * p.ldo + at(c, 0), o);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (at(c, j) < p.d) scalar_store(p.out, p.out_dtype, row * p.ldo + at(c, j), o[j]);
            }
        }
    }
    if (CODES) {
        most = __reduce_max_sync(0xffffffffu, lane < warps ? wmax[lane] : 0u);
        const bool finite = most < 0x7F800000u;
        const float s = __fdiv_rn(__uint_as_float(most), 127.f), inv = __fdiv_rn(1.f, s);
        if (tid == 0) p.scales[row] = !finite ? __uint_as_float(0x7FC00000u) : most == 0 ? 0.f : __fmul_rn(s, q);
        const bool none = !finite || most == 0;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            int k[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                // u * (1 / s) is within 2.3e-5 of u / s (127 times two roundings and the quotient's own), so that only where it is
                // next to a border the division has to be made (and where 1 / s is no number: rows below 1e-36)
                const float t = u[c][j] * inv;
                float n = rintf(t);
                if (!(fabsf(t - n) <= 0.4999f)) n = rintf(__fdiv_rn(u[c][j], s));
                k[j] = none ? 0 : max(-127, min(127, (int)n));
            }
            if (VEC) {
                if (at(c, 0) < p.d) {
                    uint2 o;
                    o.x = (uint32_t)(k[0] & 255) | (uint32_t)(k[1] & 255) << 8 | (uint32_t)(k[2] & 255) << 16 | (uint32_t)k[3] << 24;
                    o.y = (uint32_t)(k[4] & 255) | (uint32_t)(k[5] & 255) << 8 | (uint32_t)(k[6] & 255) << 16 | (uint32_t)k[7] << 24;
                    *reinterpret_cast<uint2*>(p.codes + row * p.ldc + at(c, 0)) = o;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (at(c, j) < p.d) p.codes[row * p.ldc + at(c, j)] = (int8_t)k[j];
            }
        }
    }
}

typedef void (*NormKernel)(NormParams);
template <int NCH, bool VEC>
NormKernel norm_pick(bool codes, int rotate) {
    if (!codes) return add_rmsnorm_kernel<NCH, VEC, false, 1>;
    return rotate == 256 ? add_rmsnorm_kernel<NCH, VEC, true, 256> : rotate == 32 ? add_rmsnorm_kernel<NCH, VEC, true, 32> : add_rmsnorm_kernel<NCH, VEC, true, 1>;
}
template <bool VEC>
NormKernel norm_pick(int nch, bool codes, int rotate) {
    return nch == 1 ? norm_pick<1, VEC>(codes, rotate) : nch == 2 ? norm_pick<2, VEC>(codes, rotate) : norm_pick<4, VEC>(codes, rotate);
}

bool known(int32_t dtype) { return dtype >= 0 && dtype <= 2; }
bool aligned(const void* p, int64_t ld, int esz, int to) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % to == 0 && ld * esz % to == 0);
}

}  // namespace
}  // namespace iq

using namespace iq;

extern "C" int32_t iq_add_rmsnorm(iq_ctx* ctx, void* stream, const void* x, int32_t x_dtype, int64_t ldx, const void* residual,
                                  int32_t r_dtype, int64_t ldr, void* residual_out, int64_t ldro, const void* weight, int32_t w_dtype,
                                  float weight_offset, float eps, int32_t rows, int32_t d, void* out, int32_t out_dtype, int64_t ldo,
                                  int8_t* codes, int64_t ldc, float* scales, int32_t rotate) {
    // (the checks come before the context is looked at: they are the same without a GPU)
    if (rows < 0 || d < 1 || !(eps >= 0.f)) return fail(ctx, kErrInvalidArg, "add_rmsnorm: rows = %d, d = %d, eps = %g", rows, d, (double)eps);
    if (d > kNormMaxD) return fail(ctx, kErrUnsupported, "add_rmsnorm: d = %d (up to %d)", d, kNormMaxD);
    if (residual == nullptr || !known(r_dtype) || ldr < d || (weight != nullptr && !known(w_dtype)))
        return fail(ctx, kErrInvalidArg, "add_rmsnorm: residual and weight of fp32, fp16 or bf16, rows at least d apart");
    if (x != nullptr ? !known(x_dtype) || ldx < d || residual_out == nullptr || ldro < d : residual_out != nullptr)
        return fail(ctx, kErrInvalidArg, "add_rmsnorm: x of fp32, fp16 or bf16 and a place for the sum, or neither");
    if (out == nullptr && codes == nullptr) return fail(ctx, kErrInvalidArg, "add_rmsnorm: neither out nor codes");
    if (out != nullptr && (!known(out_dtype) || ldo < d)) return fail(ctx, kErrInvalidArg, "add_rmsnorm: out of fp32, fp16 or bf16, rows at least d apart");
    if (codes != nullptr ? scales == nullptr || ldc < d : scales != nullptr)
        return fail(ctx, kErrInvalidArg, "add_rmsnorm: codes come with scales, rows at least d apart");
    if (rotate != 0 && rotate != 32 && rotate != 256) return fail(ctx, kErrUnsupported, "add_rmsnorm: rotation in blocks of %d (0, 32 or 256)", rotate);
    if (rotate != 0 && (codes == nullptr || d % rotate != 0))
        return fail(ctx, kErrInvalidArg, "add_rmsnorm: the rotation is the codes', d = %d a multiple of its blocks of %d", d, rotate);
    if (ctx == nullptr) return kErrInvalidArg;
    if (rows == 0) return kOk;
    NormParams p;
    p.x = x; p.r = residual; p.r_out = residual_out; p.w = weight; p.out = out; p.codes = codes; p.scales = scales;
    p.ldx = ldx; p.ldr = ldr; p.ldro = ldro; p.ldo = ldo; p.ldc = ldc;
    p.x_dtype = x_dtype; p.r_dtype = r_dtype; p.w_dtype = w_dtype; p.out_dtype = out_dtype;
    p.d = d; p.offset = weight_offset; p.eps = eps;
    const bool vec = d % 8 == 0 && aligned(x, ldx, dtype_size(x_dtype), 16) && aligned(residual, ldr, dtype_size(r_dtype), 16) &&
                     aligned(residual_out, ldro, dtype_size(r_dtype), 16) && aligned(weight, 0, 1, 16) && aligned(out, ldo, dtype_size(out_dtype), 16) &&
                     aligned(codes, ldc, 1, 8);
    const int groups = (d + 7) / 8, nch = groups <= 1024 ? 1 : groups <= 2048 ? 2 : 4;
    const int threads = round_up((groups + nch - 1) / nch, 32);
    const NormKernel kernel = vec ? norm_pick<true>(nch, codes != nullptr, rotate) : norm_pick<false>(nch, codes != nullptr, rotate);
    DeviceScope on(ctx);
    if (on.error != cudaSuccess) return check_cuda(ctx, on.error, "add_rmsnorm device");
    return check_cuda(ctx, launch_dependent(kernel, dim3(rows), threads, 0, reinterpret_cast<cudaStream_t>(stream), p), "add_rmsnorm launch");
}
