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

#include <algorithm>

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
    int32_t rows, d;
    float offset, eps;
};

// Eight values as they lie in memory, and as floats. A dtype is the same for a whole launch; HT is the 16-bit type where all 16-bit tensors
// of the call have the same one, else kF32: chosen at run time, where both conversions are made.
template <int HT>
__device__ __forceinline__ int32_t known_type(int32_t dtype) { return HT == kF32 || dtype == kF32 ? dtype : HT; }

struct Raw8 {
    uint4 a, b;
};
__device__ __forceinline__ Raw8 load8(const void* p, int32_t dtype, size_t i) {
    Raw8 r;
    r.b = make_uint4(0, 0, 0, 0);
    if (dtype == kF32) {
        const float* q = static_cast<const float*>(p) + i;
        asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r.a.x), "=r"(r.a.y), "=r"(r.a.z), "=r"(r.a.w), "=r"(r.b.x), "=r"(r.b.y), "=r"(r.b.z), "=r"(r.b.w)
                     : "l"(q)
                     : "memory");
    } else {
        r.a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    }
    return r;
}
template <int HT>
__device__ __forceinline__ void unpack8(const Raw8& r, int32_t dtype, float (&v)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (dtype == kF32) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = __uint_as_float(w[j]);
    } else if (known_type<HT>(dtype) == kBF16) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            v[2 * j] = __uint_as_float(w[j] << 16);
            v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
        }
    }
}
template <int HT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi, int32_t dtype) {
    if (known_type<HT>(dtype) == kF16) return pack_half2(lo, hi);
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}
// v rounded to the type, as it lies in memory; v becomes what was stored
template <int HT>
__device__ __forceinline__ Raw8 pack8(int32_t dtype, const float (&v)[8]) {
    Raw8 r;
    if (dtype == kF32) {
        r.a = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        r.b = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
        r.a = make_uint4(pack2<HT>(v[0], v[1], dtype), pack2<HT>(v[2], v[3], dtype), pack2<HT>(v[4], v[5], dtype), pack2<HT>(v[6], v[7], dtype));
        r.b = make_uint4(0, 0, 0, 0);
    }
    return r;
}
__device__ __forceinline__ void store8(void* p, int32_t dtype, size_t i, const Raw8& r) {
    if (dtype == kF32) {
        // (whole sectors: with two stores of 16 bytes, 32 apart between lanes, 4096 rows of 7680 took 2 us longer)
        asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(static_cast<float*>(p) + i), "r"(r.a.x), "r"(r.a.y), "r"(r.a.z), "r"(r.a.w),
                     "r"(r.b.x), "r"(r.b.y), "r"(r.b.z), "r"(r.b.w)
                     : "memory");
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = r.a;
    }
}
// One value at a time, for rows that are not aligned: as it lies in memory, and as a float
__device__ __forceinline__ uint32_t load1(const void* p, int32_t dtype, size_t i) {
    return dtype == kF32 ? static_cast<const uint32_t*>(p)[i] : (uint32_t)static_cast<const uint16_t*>(p)[i];
}
template <int HT>
__device__ __forceinline__ float unpack1(uint32_t v, int32_t dtype) {
    if (dtype == kF32) return __uint_as_float(v);
    return known_type<HT>(dtype) == kBF16 ? bf16_bits_to_f32(v) : __half2float(__ushort_as_half((unsigned short)v));
}
template <int HT>
__device__ __forceinline__ float round1(float v, int32_t dtype) {
    if (dtype == kF32) return v;
    return known_type<HT>(dtype) == kBF16 ? __bfloat162float(__float2bfloat16_rn(v)) : __half2float(__float2half_rn(v));
}
template <int HT>
__device__ __forceinline__ void store1(void* p, int32_t dtype, size_t i, float v) {
    if (dtype == kF32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = known_type<HT>(dtype) == kBF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}
// Largest magnitude of three, NaN if one of them is
__device__ __forceinline__ float max_abs(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float max_abs8(float m, const float (&u)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) m = max_abs(m, u[j], u[j + 1]);
    return m;
}

// Two neighbouring values per instruction, each rounded as by itself
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float lo, float hi) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void apart(Two t, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(t)); }
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
// PACKED: two per instruction. (Where the memory is the bound the moves into pairs of registers cost more than they save: 4096 rows of 4096, norm alone, 32.0 us one by
// one and 36.8 in pairs.)
template <bool PACKED>
__device__ __forceinline__ void add8(float (&a)[8], const float (&b)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        if (PACKED) {
            apart(add2(two(a[j], a[j + 1]), two(b[j], b[j + 1])), a[j], a[j + 1]);
        } else {
            a[j] = __fadd_rn(a[j], b[j]);
            a[j + 1] = __fadd_rn(a[j + 1], b[j + 1]);
        }
    }
}
template <bool PACKED>
__device__ __forceinline__ void mul8(const float (&a)[8], const float (&b)[8], float (&r)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        if (PACKED) {
            apart(mul2(two(a[j], a[j + 1]), two(b[j], b[j + 1])), r[j], r[j + 1]);
        } else {
            r[j] = __fmul_rn(a[j], b[j]);
            r[j + 1] = __fmul_rn(a[j + 1], b[j + 1]);
        }
    }
}
// The sum of eight squares: of the even ones and of the odd ones
template <bool PACKED>
__device__ __forceinline__ float squares8(const float (&v)[8]) {
    float even, odd;
    if (PACKED) {
        Two s = mul2(two(v[0], v[1]), two(v[0], v[1]));
#pragma unroll
        for (int j = 2; j < 8; j += 2) s = fma2(two(v[j], v[j + 1]), two(v[j], v[j + 1]), s);
        apart(s, even, odd);
    } else {
        even = __fmul_rn(v[0], v[0]);
        odd = __fmul_rn(v[1], v[1]);
#pragma unroll
        for (int j = 2; j < 8; j += 2) {
            even = __fmaf_rn(v[j], v[j], even);
            odd = __fmaf_rn(v[j + 1], v[j + 1], odd);
        }
    }
    return __fadd_rn(even, odd);
}

// Butterflies inside a thread, and between lanes h apart: a + b in the lower one, a - b in the upper one, one rounding each.
// a, b -> a + b, a - b (the product with -1 is exact)
__device__ __forceinline__ void butterfly2(float& a0, float& a1, float& b0, float& b1) {
    const Two a = two(a0, a1), b = two(b0, b1);
    apart(add2(a, b), a0, a1);
    apart(fma2(b, two(-1.f, -1.f), a), b0, b1);
}
// spans 1, 2 and 4
__device__ __forceinline__ void rotate_eight(float (&u)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float a = u[j], b = u[j + 1];
        u[j] = __fadd_rn(a, b);
        u[j + 1] = __fsub_rn(a, b);
    }
#pragma unroll
    for (int h = 2; h < 8; h <<= 1)
#pragma unroll
        for (int j = 0; j < 8; j += 2)
            if ((j & h) == 0) butterfly2(u[j], u[j + 1], u[j + h], u[j + h + 1]);
}
__device__ __forceinline__ void rotate_lanes(float (&u)[8], int lane, int h) {
    const float sign = (lane & h) ? -1.f : 1.f;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const Two other = two(__shfl_xor_sync(0xffffffffu, u[j], h), __shfl_xor_sync(0xffffffffu, u[j + 1], h));
        apart(fma2(two(sign, sign), two(u[j], u[j + 1]), other), u[j], u[j + 1]);
    }
}
// Blocks of ROT inputs of which a thread has eight in a row
template <int ROT>
__device__ __forceinline__ void rotate8(float (&u)[8], int lane) {
    if (ROT == 1) return;
    rotate_eight(u);
#pragma unroll
    for (int h = 1; h < ROT / 8; h <<= 1) rotate_lanes(u, lane, h);
}

// Eight codes rint(u / s), s > 0. m = u * inv + 1.5 * 2^23 holds the rounded product in its low bits. u * inv (inv = 1 / s) is within 1.6e-5 of the
// quotient as fp32 rounds it (127 times 2^-24 for inv and for the quotient), so the division itself is only made where the product is next to
// a border (or inv is no number: s below 2^-128).
__device__ __forceinline__ uint2 codes8(const float (&u)[8], float s, float inv) {
    constexpr float kMagic = 12582912.f, kFar = 0.49998f;
    uint32_t m[8];
    float off[8];
    const Two i2 = two(inv, inv), magic = two(kMagic, kMagic);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const Two v = fma2(two(u[j], u[j + 1]), i2, magic), minus_n = fma2(v, two(-1.f, -1.f), magic);
        float a, b;
        apart(v, a, b);
        m[j] = __float_as_uint(a);
        m[j + 1] = __float_as_uint(b);
        apart(fma2(two(u[j], u[j + 1]), i2, minus_n), off[j], off[j + 1]);
    }
    if (!(max_abs8(0.f, off) <= kFar)) {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (!(fabsf(fmaf(u[j], inv, kMagic - __uint_as_float(m[j]))) <= kFar)) m[j] = (uint32_t)max(-127, min(127, __float2int_rn(__fdiv_rn(u[j], s))));
    }
    return make_uint2(__byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(m[4], m[5], 0x0040), __byte_perm(m[6], m[7], 0x0040), 0x5410));
}

// A row per block, NCH times eight values per thread. Above 16,384 values (NCH = 4) 64 registers per thread do not hold the sums, weights and codes: 224 to 424 bytes of each
// thread's values lie in local memory (up to 200 where rows are not aligned, 8 to 32 with NCH = 2). One row of 16,384 in bf16 4.0 us, of 18,432 9.8, of 32,768 15.7; 1024 rows of them 23.0 (floor 20.6), 73 (23.1), 122
// (41.1), with rotated codes 28.4 (18.0), 97 (20.2), 161 (36.0), of fp16 29.0, 121, 213.
// VEC: rows of whole groups of eight that lie on their own size. Else value by value: neighbouring threads take
// neighbouring values, and where the rotation wants a thread to have eight in a row, they pass through shared memory.
// CODES, ROT: int8 codes, rotated in blocks of ROT inputs (1: not).
template <int NCH, int MAXT, bool VEC, bool CODES, int ROT, int HT>
__global__ void __launch_bounds__(MAXT, MAXT < 1024 ? (NCH == 1 ? 1536 : 1024) / MAXT : 0) add_rmsnorm_kernel(const __grid_constant__ NormParams p) {
    constexpr int PARTS = NCH * MAXT / 32;  // runs of 256 values
    __shared__ float wsum[PARTS], wmax[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const size_t row = blockIdx.x;
    pdl_launch_dependents();
    __shared__ __align__(16) float turn[VEC || ROT == 1 ? 1 : MAXT * 8];  // a warp's 256 values on their way to eight in a row per thread, and back
    auto at = [&](int c, int j) { return (c * (int)blockDim.x + warp * 32) * 8 + (VEC ? lane * 8 + j : j * 32 + lane); };
    pdl_wait();  // (the weight, too, may be what the kernel before has written: a norm's may depend on the input)
    Raw8 rw[VEC ? NCH : 1];
    float v[NCH][8];  // r'
    if (VEC) {
        Raw8 rr[NCH], xx[NCH];
#pragma unroll
        for (int c = 0; c < NCH; c++)
            if (at(c, 0) < p.d) {
                rr[c] = load8(p.r, p.r_dtype, row * p.ldr + at(c, 0));
                if (p.x != nullptr) xx[c] = load8(p.x, p.x_dtype, row * p.ldx + at(c, 0));
                if (p.w != nullptr) rw[VEC ? c : 0] = load8(p.w, p.w_dtype, at(c, 0));
            }
#pragma unroll
        for (int c = 0; c < NCH; c++) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[c][j] = 0.f;
            if (at(c, 0) < p.d) {
                unpack8<HT>(rr[c], p.r_dtype, v[c]);
                if (p.x != nullptr) {
                    float xv[8];
                    unpack8<HT>(xx[c], p.x_dtype, xv);
                    add8<false>(v[c], xv);
                    const Raw8 stored = pack8<HT>(p.r_dtype, v[c]);
                    store8(p.r_out, p.r_dtype, row * p.ldro + at(c, 0), stored);
                    unpack8<HT>(stored, p.r_dtype, v[c]);
                }
            }
        }
    } else {
        // (sixteen loads under way: the indexes are cut at the row's end, no guard stands between them)
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            uint32_t rr[8], xx[8];
#pragma unroll
            for (int j = 0; j < 8; j++) rr[j] = load1(p.r, p.r_dtype, row * p.ldr + min(at(c, j), p.d - 1));
            if (p.x != nullptr) {
#pragma unroll
                for (int j = 0; j < 8; j++) xx[j] = load1(p.x, p.x_dtype, row * p.ldx + min(at(c, j), p.d - 1));
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[c][j] = unpack1<HT>(rr[j], p.r_dtype);
                if (p.x != nullptr) v[c][j] = round1<HT>(v[c][j] + unpack1<HT>(xx[j], p.x_dtype), p.r_dtype);
                if (at(c, j) >= p.d) v[c][j] = 0.f;
            }
        }
        if (p.x != nullptr) {  // (behind all loads: r_out may be r)
#pragma unroll
            for (int c = 0; c < NCH; c++)
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (at(c, j) < p.d) store1<HT>(p.r_out, p.r_dtype, row * p.ldro + at(c, j), v[c][j]);
        }
    }
    // The squares of 256 neighbouring values are a sum of their own, and so are the sums' sum, in an order that is the same for every launch on rows that are aligned
    // (VEC here, and the kernel of many rows). Where they are not, a lane has other values of the 256: out and scales of a copy of the row may differ in the last bits.
    float sums[NCH];
#pragma unroll
    for (int c = 0; c < NCH; c++) sums[c] = squares8<false>(v[c]);
    // w + offset of the thread's values
    auto weights = [&](int c, float (&w)[8]) {
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = 1.f;
        if (p.w == nullptr) return;
        if (VEC) {
            if (at(c, 0) < p.d) unpack8<HT>(rw[VEC ? c : 0], p.w_dtype, w);
        } else {
            uint32_t ww[8];
#pragma unroll
            for (int j = 0; j < 8; j++) ww[j] = load1(p.w, p.w_dtype, min(at(c, j), p.d - 1));
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = unpack1<HT>(ww[j], p.w_dtype);
        }
#pragma unroll
        for (int j = 0; j < 8; j++) w[j] = __fadd_rn(w[j], p.offset);
    };
    float u[CODES ? NCH : 1][8];
    if (CODES) {
        float most = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            float w[8];
            weights(c, w);
            mul8<false>(v[c], w, u[c]);
            if (!VEC && ROT > 1) {
                float* const mine = turn + warp * 256;
#pragma unroll
                for (int j = 0; j < 8; j++) mine[j * 32 + lane] = u[c][j];
                __syncwarp();
                const float4 a = *reinterpret_cast<const float4*>(mine + lane * 8), b = *reinterpret_cast<const float4*>(mine + lane * 8 + 4);
                u[c][0] = a.x; u[c][1] = a.y; u[c][2] = a.z; u[c][3] = a.w;
                u[c][4] = b.x; u[c][5] = b.y; u[c][6] = b.z; u[c][7] = b.w;
                __syncwarp();
            }
            rotate8<ROT>(u[c], lane);
            most = max_abs8(most, u[c]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, most, o);
            most = max_abs(most, other, other);
        }
        if (lane == 0) wmax[warp] = most;
    }
#pragma unroll
    for (int c = 0; c < NCH; c++) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sums[c] += __shfl_xor_sync(0xffffffffu, sums[c], o);
        if (lane == 0) wsum[c * warps + warp] = sums[c];
    }
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < (PARTS + 31) / 32; c++)  // (parts beyond the row are zeros)
        if (32 * c + lane < NCH * warps) sum += wsum[32 * c + lane];
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
                if (at(c, 0) < p.d) store8(p.out, p.out_dtype, row * p.ldo + at(c, 0), pack8<HT>(p.out_dtype, o));
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (at(c, j) < p.d) store1<HT>(p.out, p.out_dtype, row * p.ldo + at(c, j), o[j]);
            }
        }
    }
    if (CODES) {
        float most = lane < warps ? wmax[lane] : 0.f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, most, o);
            most = max_abs(most, other, other);
        }
        const bool finite = most < INFINITY;  // (not with a NaN either)
        const float s = __fdiv_rn(most, 127.f), inv = __fdiv_rn(1.f, s);
        if (tid == 0) p.scales[row] = !finite ? __uint_as_float(0x7FC00000u) : s == 0.f ? 0.f : __fmul_rn(s, q);
        const bool none = !finite || s == 0.f;  // (s: a largest magnitude below 2^-143 has none either)
#pragma unroll
        for (int c = 0; c < NCH; c++) {
            const uint2 k = none ? make_uint2(0, 0) : codes8(u[c], s, inv);
            if (VEC) {
                if (at(c, 0) < p.d) *reinterpret_cast<uint2*>(p.codes + row * p.ldc + at(c, 0)) = k;
            } else if (ROT > 1) {  // codes of eight values in a row per thread, stored neighbour by neighbour
                uint2* const mine = reinterpret_cast<uint2*>(turn + warp * 256);
                mine[lane] = k;
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (at(c, j) < p.d) p.codes[row * p.ldc + at(c, j)] = reinterpret_cast<const int8_t*>(mine)[j * 32 + lane];
                __syncwarp();
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (at(c, j) < p.d) p.codes[row * p.ldc + at(c, j)] = (int8_t)((j < 4 ? k.x : k.y) >> (8 * (j & 3)));
            }
        }
    }
}

// Many rows of up to 16384: a block takes one row after the other, a warp 512 values of it: sixteen lanes share 256 of them, and a lane has two
// groups of eight, 128 apart, so that spans 8 to 64 of a rotation go from lane to lane. The next row is under way into shared memory
// meanwhile, copied by the warp that uses it, so that no barrier stands between copy and use. One barrier per row, the sums of two rows in turn.
//
// Bound: issue slots where codes are wanted (38 instructions per rotated value; operations on pairs of values saved 4 %), else the memory. 4096 rows of 4096,
// bf16 added to bf16, us, the kernel of a row per block / this one: out 27.8 / 22.9 (floor 20.5), codes 32.3 / 21.1, rotated 44.3 / 26.9 (18.0); 7680 wide
// 70 / 43.3, 80 / 37.1, 94 / 49.4. On the way: types chosen at run time 24.3, 27.6, 33.5, and addresses made per row 23.3, 29.3, 34.0; with one group
// per lane then 26.2, 33.0, 37.4, with four 27.9, 30.5, 35.3, with a third stage 25.4, 29.5, 34.3.
constexpr int kNormStages = 2;
constexpr int kNormRowsSmem = 200 * 1024;  // of an SM's blocks
// TYPES: kSum32 and kSum16 have a 16-bit x and out and a residual of fp32 or the same type; kAnyTypes asks at run time, which makes both of every
// conversion.
enum { kAnyTypes, kSum32, kSum16 };
template <int TYPES, bool OUT, bool CODES, int ROT, int HT>
__global__ void __launch_bounds__(1024) add_rmsnorm_rows_kernel(const __grid_constant__ NormParams p) {
    constexpr int K = 2, LB = 32 / K, APART = 256 / K;  // groups of a lane, lanes of 256 values, values between a lane's groups
    extern __shared__ uint4 ring[];                     // r, then x: [stage][group of the lane][warp][lane]
    __shared__ float wsum[2][64], wmax[2][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
    const int block = warp * 256 * K + (lane / LB) * 256, first = block + (lane % LB) * 8;  // the lanes' 256 values, the lane's first one
    const bool live[K] = {first < p.d, first + APART < p.d};
    pdl_launch_dependents();
    // Everything that a row's addresses are made of, once
    const int32_t r_dtype = TYPES == kAnyTypes ? p.r_dtype : TYPES == kSum32 ? kF32 : HT, x_dtype = TYPES == kAnyTypes ? p.x_dtype : HT;
    const int32_t out_dtype = TYPES == kAnyTypes ? p.out_dtype : HT;
    const bool wide_r = r_dtype == kF32, wide_x = x_dtype == kF32, add = TYPES != kAnyTypes || p.x != nullptr;
    const uint32_t r_size = wide_r ? 4 : 2, x_size = wide_x ? 4 : 2, o_size = out_dtype == kF32 ? 4 : 2;
    // a copy is 16 bytes: a group of 16-bit values; of fp32 ones LB lanes copy 16 LB neighbouring bytes twice
    struct Source {
        const char* row;
        int64_t step;         // to the block's next row
        uint32_t to, stage, group_to, group_from;
        bool first, second;   // whether the copies of the lane's first and second group lie in the row
        bool first2, second2;  // fp32: and 16 LB bytes further
    };
    auto source = [&](const void* t, int64_t ld, uint32_t size, uint32_t ring_at) {
        Source s;
        const int at = size == 4 ? block + (lane % LB) * 4 : first;
        s.row = static_cast<const char*>(t) + ((int64_t)blockIdx.x * ld + at) * size;
        s.step = (int64_t)gridDim.x * ld * size;
        s.stage = warps * 256 * K * size;
        s.group_to = warps * 256 * size;
        s.group_from = APART * size;
        s.to = ring_at + warp * 256 * size + (size == 4 ? (lane / LB) * (LB * 32) + (lane % LB) * 16 : lane * 16);
        s.first = at < p.d;
        s.second = at + APART < p.d;
        s.first2 = at + LB * 4 < p.d;
        s.second2 = at + APART + LB * 4 < p.d;
        return s;
    };
    const uint32_t base = smem_u32(ring), x_base = base + kNormStages * warps * 256 * K * r_size;
    Source r = source(p.r, p.ldr, r_size, base), x = source(p.x, p.ldx, x_size, x_base);
    uint32_t r_from = base + (warp * 32 + lane) * 8 * r_size, x_from = x_base + (warp * 32 + lane) * 8 * x_size;
    char* r_out = static_cast<char*>(p.r_out) + ((int64_t)blockIdx.x * p.ldro + first) * r_size;
    char* out = static_cast<char*>(p.out) + ((int64_t)blockIdx.x * p.ldo + first) * o_size;
    int8_t* codes = p.codes + (int64_t)blockIdx.x * p.ldc + first;
    const int64_t r_out_step = (int64_t)gridDim.x * p.ldro * r_size, out_step = (int64_t)gridDim.x * p.ldo * o_size, codes_step = (int64_t)gridDim.x * p.ldc;
    auto copy = [&](Source& s, bool wide, uint32_t to) {
        if (s.first) cp_async_cg16(to, s.row);
        if (s.second) cp_async_cg16(to + s.group_to, s.row + s.group_from);
        if (wide) {
            if (s.first2) cp_async_cg16(to + LB * 16, s.row + LB * 16);
            if (s.second2) cp_async_cg16(to + s.group_to + LB * 16, s.row + s.group_from + LB * 16);
        }
        s.row += s.step;
    };
    auto take = [&](uint32_t from, bool wide) {
        Raw8 v;
        v.a = lds128(from);
        v.b = wide ? lds128(from + 16) : make_uint4(0, 0, 0, 0);
        return v;
    };
    pdl_wait();
    static_assert(kNormStages == 2, "a stage for the row under work and one for the next");
    copy(r, wide_r, r.to);  // (there are no more blocks than rows)
    if (add) copy(x, wide_x, x.to);
    asm volatile("cp.async.commit_group;" ::: "memory");
    float w[K][8];
#pragma unroll
    for (int k = 0; k < K; k++) {
#pragma unroll
        for (int j = 0; j < 8; j++) w[k][j] = 1.f;
        if (p.w != nullptr && live[k]) {
            unpack8<HT>(load8(p.w, p.w_dtype, first + APART * k), p.w_dtype, w[k]);
#pragma unroll
            for (int j = 0; j < 8; j++) w[k][j] = __fadd_rn(w[k][j], p.offset);
        }
    }
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        // the next row, into the stage of the row before: a barrier has passed since it was read
        const uint32_t r_at = turn ? r.stage : 0, x_at = turn ? x.stage : 0;
        if (row + gridDim.x < p.rows) {
            copy(r, wide_r, r.to + (r.stage - r_at));
            if (add) copy(x, wide_x, x.to + (x.stage - x_at));
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncwarp();
        float v[K][8], sums[K];
#pragma unroll
        for (int k = 0; k < K; k++) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[k][j] = 0.f;
            if (live[k]) {
                unpack8<HT>(take(r_from + r_at + k * r.group_to, wide_r), r_dtype, v[k]);
                if (add) {
                    float xv[8];
                    unpack8<HT>(take(x_from + x_at + k * x.group_to, wide_x), x_dtype, xv);
                    add8<CODES>(v[k], xv);
                    const Raw8 stored = pack8<HT>(r_dtype, v[k]);
                    store8(r_out + k * r.group_from, r_dtype, 0, stored);
                    if (!wide_r) unpack8<HT>(stored, r_dtype, v[k]);
                }
            }
            sums[k] = squares8<CODES>(v[k]);
        }
        r_out += r_out_step;
        // (the order of the other kernel's lanes: 16, 8, 4, 2 and 1 groups apart)
        float sum = sums[0] + sums[1];
#pragma unroll
        for (int o = LB / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane % LB == 0) wsum[turn][warp * K + lane / LB] = sum;
        float most = 0.f;
        float kept[OUT && CODES ? K : 1][8];  // r', where both outputs are wanted; v is u from here on
        if (CODES) {
#pragma unroll
            for (int k = 0; k < K; k++) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (OUT) kept[OUT ? k : 0][j] = v[k][j];
                mul8<true>(v[k], w[k], v[k]);
            }
            if (ROT > 1) {
#pragma unroll
                for (int k = 0; k < K; k++) {
                    rotate_eight(v[k]);
#pragma unroll
                    for (int h = 1; h < (ROT < APART ? ROT / 8 : LB); h <<= 1) rotate_lanes(v[k], lane, h);
                }
                if (ROT > APART) {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) butterfly2(v[0][j], v[0][j + 1], v[1][j], v[1][j + 1]);
                }
            }
#pragma unroll
            for (int k = 0; k < K; k++)
                most = max_abs8(most, v[k]);
            const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(most));  // (bits order as the values do, NaN last)
            if (lane == 0) wmax[turn][warp] = __uint_as_float(m);
        }
        __syncthreads();
        sum = lane < K * warps ? wsum[turn][lane] : 0.f;
        if (32 + lane < K * warps) sum += wsum[turn][32 + lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float q = rsqrtf(__fadd_rn(__fdiv_rn(sum, (float)p.d), p.eps));
        if (OUT) {
#pragma unroll
            for (int k = 0; k < K; k++)
                if (live[k]) {
                    float o[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j] = ((CODES ? kept[OUT && CODES ? k : 0][j] : v[k][j]) * q) * w[k][j];
                    store8(out + k * APART * o_size, out_dtype, 0, pack8<HT>(out_dtype, o));
                }
            out += out_step;
        }
        if (CODES) {
            most = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < warps ? __float_as_uint(wmax[turn][lane]) : 0u));
            const bool finite = most < INFINITY;  // (not with a NaN either)
            const float step = __fdiv_rn(most, 127.f), inv = __fdiv_rn(1.f, step);
            const bool none = !finite || step == 0.f;
            if (tid == 0) p.scales[row] = !finite ? __uint_as_float(0x7FC00000u) : step == 0.f ? 0.f : __fmul_rn(step, q);
#pragma unroll
            for (int k = 0; k < K; k++)
                if (live[k]) *reinterpret_cast<uint2*>(codes + k * APART) = none ? make_uint2(0, 0) : codes8(v[k], step, inv);
            codes += codes_step;
        }
        turn ^= 1;
    }
}

// (Of the kernel of many rows 16 to 32 bytes per thread lie in local memory where codes are wanted, 56 where out is as well and the types are chosen at run time: 4096 rows
// of 4096, bf16, rotated codes 27.0 us, with out 30.8 (floors 18.0 and 23.1); fp32 throughout 39.0 and 62.7 (33.4 and 43.7).)
typedef void (*NormKernel)(NormParams);
template <int TYPES, int HT>
NormKernel norm_pick_rows(bool out, bool codes, int rotate) {
    if (!codes) return add_rmsnorm_rows_kernel<TYPES, true, false, 1, HT>;
    if (out)
        return rotate == 256 ? add_rmsnorm_rows_kernel<TYPES, true, true, 256, HT> : rotate == 32 ? add_rmsnorm_rows_kernel<TYPES, true, true, 32, HT>
                                                                                               : add_rmsnorm_rows_kernel<TYPES, true, true, 1, HT>;
    return rotate == 256 ? add_rmsnorm_rows_kernel<TYPES, false, true, 256, HT> : rotate == 32 ? add_rmsnorm_rows_kernel<TYPES, false, true, 32, HT>
                                                                                            : add_rmsnorm_rows_kernel<TYPES, false, true, 1, HT>;
}
template <int HT>
NormKernel norm_pick_rows(int types, bool out, bool codes, int rotate) {
    return types == kSum32 ? norm_pick_rows<kSum32, HT>(out, codes, rotate) : types == kSum16 ? norm_pick_rows<kSum16, HT>(out, codes, rotate)
                                                                                             : norm_pick_rows<kAnyTypes, HT>(out, codes, rotate);
}
NormKernel norm_pick_rows(int half, int types, bool out, bool codes, int rotate) {
    return half == kF16 ? norm_pick_rows<kF16>(types, out, codes, rotate) : half == kBF16 ? norm_pick_rows<kBF16>(types, out, codes, rotate)
                                                                                         : norm_pick_rows<kAnyTypes, kF32>(out, codes, rotate);
}
template <int NCH, int MAXT, bool VEC, int HT>
NormKernel norm_pick(bool codes, int rotate) {
    if (!codes) return add_rmsnorm_kernel<NCH, MAXT, VEC, false, 1, HT>;
    return rotate == 256 ? add_rmsnorm_kernel<NCH, MAXT, VEC, true, 256, HT> : rotate == 32 ? add_rmsnorm_kernel<NCH, MAXT, VEC, true, 32, HT>
                                                                                            : add_rmsnorm_kernel<NCH, MAXT, VEC, true, 1, HT>;
}
template <int NCH>
NormKernel norm_pick(int half, bool codes, int rotate) {
    return half == kF16 ? norm_pick<NCH, 1024, true, kF16>(codes, rotate) : half == kBF16 ? norm_pick<NCH, 1024, true, kBF16>(codes, rotate)
                                                                                          : norm_pick<NCH, 1024, true, kF32>(codes, rotate);
}
// Rows that are not aligned: blocks of up to 512 threads, whose registers are held to what lets 1536 of them (with two groups each 1024) share an SM: more rows under
// way at once. 2048 rows of 4095, bf16, 27.0 -> 22.4 us, with the one 16-bit type known 20.8; 1024 of 7681 29.9 -> 26.1 -> 22.3; 30,000 of 480 with rotated codes
// 113 -> 55 -> 51. Up to a row per SM (few) a thread per group: 113 of 7680 5.5 -> 3.9. Taken back: groups of eight out of aligned pieces of 16 bytes, shifted in registers (2048 rows of 4095 33.0).
template <int HT>
NormKernel norm_pick_unaligned(int groups, bool few, bool codes, int rotate) {
    return groups <= 256 ? norm_pick<1, 256, false, HT>(codes, rotate) : groups <= 512 ? norm_pick<1, 512, false, HT>(codes, rotate)
         : groups <= 1024 && few ? norm_pick<1, 1024, false, HT>(codes, rotate) : groups <= 1024 ? norm_pick<2, 512, false, HT>(codes, rotate) : groups <= 2048 ? norm_pick<2, 1024, false, HT>(codes, rotate)
                                                                                        : norm_pick<4, 1024, false, HT>(codes, rotate);
}
NormKernel norm_pick_unaligned(int half, int groups, bool few, bool codes, int rotate) {
    return half == kF16 ? norm_pick_unaligned<kF16>(groups, few, codes, rotate) : half == kBF16 ? norm_pick_unaligned<kBF16>(groups, few, codes, rotate)
                                                                                                : norm_pick_unaligned<kF32>(groups, few, codes, rotate);
}

bool misplaced(const void* p, int esz) { return reinterpret_cast<uintptr_t>(p) % esz != 0; }
bool known(int32_t dtype) { return dtype >= 0 && dtype <= 2; }
// whether every group of eight of the rows lies on its own size
bool aligned(const void* p, int64_t ld, int esz) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (8 * esz) == 0 && ld % 8 == 0);
}

}  // namespace

int32_t norm_init(iq_ctx* ctx) {
    for (int half = 0; half < 3; half++)
        for (int mode = 0; mode < 21; mode++) {  // of three types: out; out and codes of three rotations; codes of three
            const int m = mode % 7;
            const NormKernel k = norm_pick_rows(half, mode / 7, m < 4, m != 0, m % 3 == 2 ? 32 : m % 3 == 0 ? 256 : 0);
            const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(k), cudaFuncAttributeMaxDynamicSharedMemorySize, kNormRowsSmem);
            if (e != cudaSuccess) return check_cuda(ctx, e, "cudaFuncSetAttribute(add_rmsnorm_rows)");
        }
    return kOk;
}

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
    if (misplaced(residual, dtype_size(r_dtype)) || misplaced(residual_out, dtype_size(r_dtype)) || (x != nullptr && misplaced(x, dtype_size(x_dtype))) ||
        (weight != nullptr && misplaced(weight, dtype_size(w_dtype))) || (out != nullptr && misplaced(out, dtype_size(out_dtype))) || misplaced(scales, 4))
        return fail(ctx, kErrInvalidArg, "add_rmsnorm: a tensor does not begin on an element");
    if (rotate != 0 && rotate != 32 && rotate != 256) return fail(ctx, kErrUnsupported, "add_rmsnorm: rotation in blocks of %d (0, 32 or 256)", rotate);
    if (rotate != 0 && (codes == nullptr || d % rotate != 0))
        return fail(ctx, kErrInvalidArg, "add_rmsnorm: the rotation is the codes', d = %d a multiple of its blocks of %d", d, rotate);
    if (ctx == nullptr) return kErrInvalidArg;
    if (rows == 0) return kOk;
    NormParams p;
    p.x = x; p.r = residual; p.r_out = residual_out; p.w = weight; p.out = out; p.codes = codes; p.scales = scales;
    p.ldx = ldx; p.ldr = ldr; p.ldro = ldro; p.ldo = ldo; p.ldc = ldc;
    p.x_dtype = x_dtype; p.r_dtype = r_dtype; p.w_dtype = w_dtype; p.out_dtype = out_dtype;
    p.rows = rows; p.d = d; p.offset = weight_offset; p.eps = eps;
    const bool vec = d % 8 == 0 && aligned(x, ldx, dtype_size(x_dtype)) && aligned(residual, ldr, dtype_size(r_dtype)) && aligned(residual_out, ldro, dtype_size(r_dtype)) &&
                     aligned(weight, 0, dtype_size(w_dtype)) && aligned(out, ldo, dtype_size(out_dtype)) && aligned(codes, ldc, 1);
    const bool few = rows <= ctx->sms;  // a block per SM: with as many threads as there are groups
    const int groups = (d + 7) / 8, nch = groups <= (vec || few ? 1024 : 512) ? 1 : groups <= 2048 ? 2 : 4;
    int threads = round_up((groups + nch - 1) / nch, 32), blocks = rows;
    size_t smem = 0;
    // the one 16-bit type of the call (bf16 where it has none), kF32 where it has both
    int half = -1;
    auto meet = [&](const void* t, int32_t dtype) {
        if (t != nullptr && dtype != kF32) half = half == -1 || half == dtype ? dtype : kF32;
    };
    meet(x, x_dtype); meet(residual, r_dtype); meet(weight, w_dtype); meet(out, out_dtype);
    if (half == -1) half = kBF16;
    const bool c8 = codes != nullptr;
    NormKernel kernel = !vec ? norm_pick_unaligned(half, groups, few, c8, rotate) : nch == 1 ? norm_pick<1>(half, c8, rotate) : nch == 2 ? norm_pick<2>(half, c8, rotate)
                                                                                                                          : norm_pick<4>(half, c8, rotate);
    // Many rows: a third more than the other kernel runs at once (64 registers a thread). 512 rows of 4096, codes of a bf16 sum, 6.8 us there and 5.2 here, 257 rows
    // 3.9 and 4.8; 200 of 7680 6.9 and 5.1, 148 3.9 and 3.6; 600 of 2048 4.4 and 4.9, 1000 5.7 and 5.2. Blocks: those that run at once, by registers and by the
    // stages in shared memory. The norm alone of an fp32 sum is at the memory's
    // rate with a row per block as well up to some 5000 values (4096 rows of 4096: 31.9 us, floor 30.8; of 7680 75 us, here 64).
    const int row_threads = (d + 511) / 512 * 32;
    const size_t row_smem = (size_t)kNormStages * row_threads * 16 * (dtype_size(r_dtype) + (x == nullptr ? 0 : dtype_size(x_dtype)));
    const int at_once = row_threads > 1024 ? 0 : ctx->sms * (int)std::min<size_t>({(size_t)(1024 / row_threads), kNormRowsSmem / row_smem, 16});
    if (vec && at_once > 0 && rows > ctx->sms * std::max(1024 / threads, 1) * 4 / 3 && (c8 || r_dtype != kF32 || d > 5120)) {
        const bool x16 = x != nullptr && x_dtype != kF32 && (out == nullptr || out_dtype != kF32);
        kernel = norm_pick_rows(half, !x16 ? kAnyTypes : r_dtype == kF32 ? kSum32 : kSum16, out != nullptr, c8, rotate);
        threads = row_threads;
        blocks = std::min(rows, at_once);
        smem = row_smem;
    }
    DeviceScope on(ctx);
    if (on.error != cudaSuccess) return check_cuda(ctx, on.error, "add_rmsnorm device");
    return check_cuda(ctx, launch_dependent(kernel, dim3(blocks), threads, smem, reinterpret_cast<cudaStream_t>(stream), p), "add_rmsnorm launch");
}
