// The sampler's rules on logits, between the lm_head and arg-max or candidates: penalties of tokens that a conversation holds already,
// biases of single tokens, and a grammar's mask.
//
//   c = how often t was generated, seen = t stands in the prompt or was generated
//   l = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   l = (l - frequency * c) - (c > 0 ? presence : 0)
//   l = l + the biases listed for t, in their order
//   out = allowed(t) ? l : -infinity
//
// The history is the row's list of tokens as the conversation has it: nothing is kept between calls. A row is a cluster's: its blocks hold a
// counter for every token of their part of the vocabulary in shared memory, read a share of the list each and count into each other's
// memory, so that the list is read once and a token's counter is where its logit is handled.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "internal.h"
#include "ptx.cuh"

namespace iq {
namespace {

constexpr int kRuleThreads = 512;
constexpr int kRuleMaxVocab = 262144;
constexpr int kRuleParts = 8;      // blocks of a row
constexpr int kRuleList = 1024;    // biases of a block's part that are added on the way; more are added behind it
constexpr int kRuleAhead = 4;      // times four logits of a thread that are under way while the history is counted
constexpr uint32_t kPrompt = 0x80000000u;

struct RuleParams {
    const void* x;
    int64_t ldx;
    float* out;
    int64_t ldo;
    int32_t x_dtype, vocab, span;  // span: logits of a block, a multiple of 128
    iq_logit_rules r;
};

__device__ __forceinline__ void red_add_cluster(uint32_t local, uint32_t cta, uint32_t v) {
    asm volatile("{\n.reg .b32 a;\nmapa.shared::cluster.u32 a, %0, %1;\nred.relaxed.cluster.shared::cluster.add.u32 [a], %2;\n}\n" ::"r"(local), "r"(cta), "r"(v) : "memory");
}
__device__ __forceinline__ void red_or_cluster(uint32_t local, uint32_t cta, uint32_t v) {
    asm volatile("{\n.reg .b32 a;\nmapa.shared::cluster.u32 a, %0, %1;\nred.relaxed.cluster.shared::cluster.or.b32 [a], %2;\n}\n" ::"r"(local), "r"(cta), "r"(v) : "memory");
}

// HIST: with counters (a cluster per row). VEC: rows of x and out lie on groups of four.
template <bool HIST, bool VEC>
__global__ void __launch_bounds__(kRuleThreads, 2) logit_rules_kernel(const __grid_constant__ RuleParams p) {
    extern __shared__ uint4 smem[];
    __shared__ int listed, rest;  // biases in the list; where the row's biases go on that found no place in it
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / kRuleParts, part = blockIdx.x % kRuleParts;
    const int lo = part * p.span, n = max(0, min(p.span, p.vocab - lo));  // this block's logits
    uint32_t* const flag = reinterpret_cast<uint32_t*>(smem);             // [span / 32] tokens that have a bias
    int* const list_t = reinterpret_cast<int*>(flag + p.span / 32);       // [kRuleList] tokens, from lo on
    float* const list_v = reinterpret_cast<float*>(list_t + kRuleList);
    uint32_t* const count = reinterpret_cast<uint32_t*>(list_v + kRuleList);  // [span]
    pdl_launch_dependents();
    for (int i = tid; i < p.span / 32; i += kRuleThreads) flag[i] = 0;
    if (HIST)
        for (int i = tid; i < p.span / 4; i += kRuleThreads) reinterpret_cast<uint4*>(count)[i] = make_uint4(0, 0, 0, 0);
    pdl_wait();
    const char* const xr = static_cast<const char*>(p.x) + (size_t)row * p.ldx * (p.x_dtype == kF32 ? 4 : 2);
    float* const out = p.out + (size_t)row * p.ldo;
    const float rep = p.r.repetition != nullptr ? p.r.repetition[row] : 1.f, pres = p.r.presence != nullptr ? p.r.presence[row] : 0.f;
    const float freq = p.r.frequency != nullptr ? p.r.frequency[row] : 0.f;
    const int m = p.r.mask == nullptr ? -1 : p.r.mask_rows != nullptr ? p.r.mask_rows[row] : row;
    const uint32_t* const mask = m >= 0 && m < p.r.masks ? p.r.mask + (size_t)m * p.r.ld_mask : nullptr;
    // four logits and their mask bits
    struct Four {
        uint4 v;
        uint32_t bits;
    };
    auto load = [&](int i) {
        Four f;
        f.v = make_uint4(0, 0, 0, 0);
        f.bits = 15;
        if (i >= n) return f;
        const int t = lo + i;
        if (VEC && i + 4 <= n) {
            if (p.x_dtype == kF32) {
                f.v = *reinterpret_cast<const uint4*>(xr + (size_t)t * 4);
            } else {
                const uint2 h = *reinterpret_cast<const uint2*>(xr + (size_t)t * 2);
                f.v.x = h.x;
                f.v.y = h.y;
            }
        } else if (p.x_dtype == kF32) {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(xr) + t;
            f.v.x = q[0];
            if (i + 1 < n) f.v.y = q[1];
            if (i + 2 < n) f.v.z = q[2];
            if (i + 3 < n) f.v.w = q[3];
        } else {
            const uint16_t* q = reinterpret_cast<const uint16_t*>(xr) + t;
            f.v.x = q[0] | (i + 1 < n ? (uint32_t)q[1] << 16 : 0u);
            f.v.y = (i + 2 < n ? q[2] : 0u) | (i + 3 < n ? (uint32_t)q[3] << 16 : 0u);
        }
        if (mask != nullptr) f.bits = mask[t >> 5] >> (t & 31) & 15u;
        return f;
    };
    Four ahead[kRuleAhead];
#pragma unroll
    for (int k = 0; k < kRuleAhead; k++) ahead[k] = load((k * kRuleThreads + tid) * 4);

    bool counts = false;
    if (HIST) {
        const int len = min(max(p.r.lens[row], 0), p.r.max_tokens);
        counts = len > 0 && (rep != 1.f || pres != 0.f || freq != 0.f);  // the same for the cluster
        if (counts) {
            const int prompt = p.r.prompt_lens != nullptr ? min(max(p.r.prompt_lens[row], 0), len) : 0;
            const int32_t* const tokens = p.r.tokens + (size_t)row * p.r.ld_tokens;
            cluster_sync_all();  // all counters are zero
            const uint32_t base = smem_u32(count);
            for (int i = part * kRuleThreads + tid; i < len; i += kRuleParts * kRuleThreads) {
                const uint32_t t = (uint32_t)tokens[i];
                if (t < (uint32_t)p.vocab) {
                    const uint32_t owner = t / (uint32_t)p.span, at = base + (t - owner * p.span) * 4;
                    if (i < prompt) red_or_cluster(at, owner, kPrompt);
                    else red_add_cluster(at, owner, 1u);
                }
            }
        }
    }
    // the biases of this block's tokens, in their order, by the last warp
    const bool biases = p.r.bias_offsets != nullptr;
    int b0 = 0, b1 = 0;
    if (biases) {
        b0 = min(max(p.r.bias_offsets[row], 0), p.r.biases);
        b1 = min(p.r.bias_offsets[row + 1], p.r.biases);
        __syncthreads();  // the flags are zero
        if (warp == kRuleThreads / 32 - 1) {
            int have = 0, j0 = b0;
            for (; j0 < b1 && have + 32 <= kRuleList; j0 += 32) {
                const uint32_t t = j0 + lane < b1 ? (uint32_t)p.r.bias_tokens[j0 + lane] - (uint32_t)lo : 0xFFFFFFFFu;
                const bool mine = t < (uint32_t)n;
                const uint32_t who = __ballot_sync(0xffffffffu, mine);
                if (mine) {
                    const int at = have + __popc(who & ((1u << lane) - 1u));
                    list_t[at] = (int)t;
                    list_v[at] = p.r.bias_values[j0 + lane];
                    atomicOr(&flag[t >> 5], 1u << (t & 31));
                }
                have += __popc(who);
            }
            if (lane == 0) {
                listed = have;
                rest = j0;
            }
        }
        __syncthreads();
    }
    if (HIST && counts) cluster_sync_all();  // every token is counted

    auto one = [&](float l, uint32_t c) {
        if (c != 0) l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
        const uint32_t said = c & ~kPrompt;
        l = __fsub_rn(l, __fmul_rn(freq, (float)said));
        return said != 0 ? __fsub_rn(l, pres) : l;
    };
    auto finish = [&](int i, const Four& f) {
        if (i >= n) return;
        float v[4];
        if (p.x_dtype == kF32) {
            v[0] = __uint_as_float(f.v.x); v[1] = __uint_as_float(f.v.y); v[2] = __uint_as_float(f.v.z); v[3] = __uint_as_float(f.v.w);
        } else if (p.x_dtype == kBF16) {
            v[0] = __uint_as_float(f.v.x << 16); v[1] = __uint_as_float(f.v.x & 0xFFFF0000u); v[2] = __uint_as_float(f.v.y << 16); v[3] = __uint_as_float(f.v.y & 0xFFFF0000u);
        } else {
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&f.v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&f.v.y));
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
        }
        if (HIST && counts) {
            const uint4 c = *reinterpret_cast<const uint4*>(count + i);
            if ((c.x | c.y | c.z | c.w) != 0) {
                if (c.x != 0) v[0] = one(v[0], c.x);
                if (c.y != 0) v[1] = one(v[1], c.y);
                if (c.z != 0) v[2] = one(v[2], c.z);
                if (c.w != 0) v[3] = one(v[3], c.w);
            }
        }
        if (biases) {
            const uint32_t has = flag[i >> 5] >> (i & 31) & 15u;
            if (has != 0) {
                const int end = listed;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (has >> j & 1)
                        for (int e = 0; e < end; e++)
                            if (list_t[e] == i + j) v[j] = __fadd_rn(v[j], list_v[e]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (!(f.bits >> j & 1)) v[j] = -INFINITY;
        if (VEC && i + 4 <= n) {
            *reinterpret_cast<float4*>(out + lo + i) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < n) out[lo + i + j] = v[j];
        }
    };
    for (int i0 = 0; i0 < n; i0 += 4 * kRuleThreads * kRuleAhead) {
#pragma unroll
        for (int k = 0; k < kRuleAhead; k++) {
            const int i = i0 + (k * kRuleThreads + tid) * 4;
            const Four f = ahead[k];
            ahead[k] = load(i + 4 * kRuleThreads * kRuleAhead);
            finish(i, f);
        }
    }
    if (biases && rest < b1) {  // more than the list holds: one after the other
        __syncthreads();
        if (warp == 0)
            for (int j = rest; j < b1; j++) {
                const uint32_t t = (uint32_t)p.r.bias_tokens[j] - (uint32_t)lo;
                if (lane == 0 && t < (uint32_t)n && (mask == nullptr || (mask[(lo + t) >> 5] >> ((lo + t) & 31) & 1)))
                    out[lo + t] = __fadd_rn(out[lo + t], p.r.bias_values[j]);
            }
    }
}

size_t rule_smem(int span, bool hist) { return (size_t)span / 8 + kRuleList * 8 + (hist ? (size_t)span * 4 : 0); }
int rule_span(int vocab) { return round_up((vocab + kRuleParts - 1) / kRuleParts, 128); }

}  // namespace

int32_t rules_init(iq_ctx* ctx) {
    const int most = (int)rule_smem(rule_span(kRuleMaxVocab), true);
    cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(logit_rules_kernel<true, true>), cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(reinterpret_cast<const void*>(logit_rules_kernel<true, false>), cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    return check_cuda(ctx, e, "cudaFuncSetAttribute(logit_rules)");
}

}  // namespace iq

using namespace iq;

extern "C" int32_t iq_logits_rules(iq_ctx* ctx, void* stream, const void* x, int32_t x_dtype, int64_t ldx, float* out, int64_t ldo, int32_t rows, int32_t vocab,
                                   const iq_logit_rules* rules) {
    // (the checks come before the context is looked at: they are the same without a GPU)
    if (x == nullptr || out == nullptr || rules == nullptr || x_dtype < 0 || x_dtype > 2) return fail(ctx, kErrInvalidArg, "logits_rules: null pointer, or x is not of fp32, fp16 or bf16");
    if (rows < 0 || vocab < 1 || ldx < vocab || ldo < vocab) return fail(ctx, kErrInvalidArg, "logits_rules: rows = %d, vocab = %d, rows at least vocab apart", rows, vocab);
    if (vocab > kRuleMaxVocab || rows > (1 << 27)) return fail(ctx, kErrUnsupported, "logits_rules: up to %d logits per row", kRuleMaxVocab);
    const iq_logit_rules& r = *rules;
    if (r.tokens != nullptr && (r.lens == nullptr || r.max_tokens < 0 || r.ld_tokens < r.max_tokens))
        return fail(ctx, kErrInvalidArg, "logits_rules: a history has lengths, its rows at least max_tokens apart");
    if (r.bias_offsets != nullptr && (r.biases < 0 || (r.biases > 0 && (r.bias_tokens == nullptr || r.bias_values == nullptr))))
        return fail(ctx, kErrInvalidArg, "logits_rules: biases are offsets, tokens and values");
    if (r.mask != nullptr && (r.masks < 1 || r.ld_mask < (vocab + 31) / 32 || (r.mask_rows == nullptr && r.masks < rows)))
        return fail(ctx, kErrInvalidArg, "logits_rules: a mask per row or mask_rows, of at least %d words", (vocab + 31) / 32);
    if (ctx == nullptr) return kErrInvalidArg;
    if (rows == 0) return kOk;
    RuleParams p;
    p.x = x; p.ldx = ldx; p.out = out; p.ldo = ldo; p.x_dtype = x_dtype; p.vocab = vocab; p.span = rule_span(vocab); p.r = r;
    const bool hist = r.tokens != nullptr && r.max_tokens > 0 && (r.repetition != nullptr || r.presence != nullptr || r.frequency != nullptr);
    const int esz = dtype_size(x_dtype);
    const bool vec = reinterpret_cast<uintptr_t>(x) % (4 * esz) == 0 && ldx % 4 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 && ldo % 4 == 0;
    auto kernel = hist ? (vec ? logit_rules_kernel<true, true> : logit_rules_kernel<true, false>) : vec ? logit_rules_kernel<false, true> : logit_rules_kernel<false, false>;
    DeviceScope on(ctx);
    if (on.error != cudaSuccess) return check_cuda(ctx, on.error, "logits_rules device");
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)rows * kRuleParts, 1, 1);
    cfg.blockDim = dim3(kRuleThreads, 1, 1);
    cfg.dynamicSmemBytes = rule_smem(p.span, hist);
    cfg.stream = reinterpret_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kRuleParts; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = hist ? 2 : 1;
    return check_cuda(ctx, cudaLaunchKernelEx(&cfg, kernel, p), "logits_rules launch");
}
