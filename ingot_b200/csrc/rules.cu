// The sampler's rules on logits, between the lm_head and arg-max or candidates: penalties of tokens that a conversation holds already,
// biases of single tokens, and a grammar's mask.
//
//   c = how often t was generated, seen = t stands in the prompt or was generated
//   l = seen ? (x > 0 ? x / repetition : x * repetition) : x
//   l = (l - frequency * c) - (c > 0 ? presence : 0)
//   l = l + the biases listed for t, in their order
//   out = allowed(t) ? l : -infinity
//
// The history is the row's list of tokens as the conversation has it: nothing is kept between calls. A block has a part of a row and a
// counter for each of its tokens in shared memory, and looks through the row's list for them.
//
// Bound: start and latencies for few rows (one of 128,000 with 2048 tokens, biases and a grammar 3.2 us), the memory for many (64 of 262,144 in fp32 without history
// 22.3 us, floor 20.6), the tokens of long histories, at which each of a row's blocks looks. Eight rows of 151,665 take 2.6 us without a history, 3.4 with one
// of no length (counters, barriers), 4.6 with 16,384 tokens of which no block has any (the looks: 13 instructions for 32, in dependent rounds), 6.6 with tokens
// spread over the vocabulary (additions to counters in shared memory, penalties), 7.0 with frequent ones and 8.1 with one alone (additions to the same
// counter). Measured and taken back: a cluster per row whose blocks share the list and count into each other's memory (11.3 us for the one row, 102 for 64 with
// 16,384 tokens against 40), parts of every so many-th run of 128 tokens instead of neighbouring ones (10.1 -> 14.6), lanes with the same token found by match
// (16.8), tokens queued until there are 32 (14.4), the next tokens loaded ahead (6.6 -> 6.9).
// A bit per token tells whether a list names one twice, which is rare: without it every bias was looked for among all (three rows of 2802 with 300 biases
// 9.7 us, now 2.1). 64 rows of 262,144 in bf16: 17.4 us without rules, 18.7 under grammars, 18.9 with 300 biases, 22.5 with 2048 tokens each, 27.6 with those and
// grammars, 28.7 with all three (floor 15.6).
#include <math.h>
#include <algorithm>
#include <type_traits>

#include "internal.h"
#include "ptx.cuh"

namespace iq {
namespace {

constexpr int kRuleMaxVocab = 262144;
constexpr int kRuleMaxTokens = 1 << 30;  // of a row's history: the steps through it stay within 32 bits
constexpr int kRulePerSm = 3;     // blocks of an SM, of 512 threads each (two with 32-bit counters of some 17,000 logits or more); one of 1024 where that is all
constexpr int kRuleSpan = 24576;  // most logits of a block,
constexpr int kRuleWhole = 32768;  // of one with an SM to itself,
constexpr int kRuleLeast = 2048;   // and least
constexpr int kRuleLook = 4;      // tokens of the history likewise, before its length is known

struct RuleParams {
    const void* x;
    int64_t ldx;
    float* out;
    int64_t ldo;
    int32_t vocab, span, parts;  // span: logits of a block, a multiple of 128; parts: blocks of a row
    uint32_t misplaced;  // elements by which x begins behind a group of eight
    iq_logit_rules r;
};

// A token's counter: how often it was generated, and on top of it whether it stands in the prompt. Two of 16 bits in a word where the history
// holds at most 32,767 tokens, else 32 bits each.
template <bool WIDE>
struct Counter {
    static constexpr uint32_t PROMPT = WIDE ? 0x80000000u : 0x8000u;
    static __device__ __forceinline__ void note(uint32_t* c, uint32_t t, bool prompt) {
        uint32_t* const w = c + (WIDE ? t : t >> 1);
        const uint32_t up = WIDE ? 0 : 16 * (t & 1);
        if (prompt) atomicOr(w, PROMPT << up);
        else atomicAdd(w, 1u << up);
    }
    static __device__ __forceinline__ uint32_t one(const uint32_t* c, uint32_t t) { return WIDE ? c[t] : reinterpret_cast<const uint16_t*>(c)[t]; }
    // the same without a branch, where t is one of n tokens
    template <bool ASKED>
    static __device__ __forceinline__ void note_if(uint32_t c, uint32_t t, uint32_t n) {
        const uint32_t at = c + (WIDE ? t * 4 : (t >> 1) * 4), v = (ASKED ? PROMPT : 1u) << (WIDE ? 0 : 16 * (t & 1));
        if (ASKED) asm volatile("{\n.reg .pred p;\nsetp.lt.u32 p, %0, %1;\n@p red.shared.or.b32 [%2], %3;\n}\n" ::"r"(t), "r"(n), "r"(at), "r"(v) : "memory");
        else asm volatile("{\n.reg .pred p;\nsetp.lt.u32 p, %0, %1;\n@p red.shared.add.u32 [%2], %3;\n}\n" ::"r"(t), "r"(n), "r"(at), "r"(v) : "memory");
    }
    // of G tokens, from i on; whether there is one
    template <int G>
    static __device__ __forceinline__ bool group(const uint32_t* c, int i, uint32_t (&r)[G]) {
        constexpr int N = WIDE ? G : G / 2;  // words
        uint32_t w[N], any = 0;
#pragma unroll
        for (int j = 0; j < N; j += N < 4 ? 2 : 4) {
            if (N < 4) {
                const uint2 a = *reinterpret_cast<const uint2*>(c + (WIDE ? i : i / 2) + j);
                w[j] = a.x; w[j + 1] = a.y;
                any |= a.x | a.y;
            } else {
                const uint4 a = *reinterpret_cast<const uint4*>(c + (WIDE ? i : i / 2) + j);
                w[j] = a.x; w[j + 1] = a.y; w[N < 4 ? 0 : j + 2] = a.z; w[N < 4 ? 0 : j + 3] = a.w;
                any |= a.x | a.y | a.z | a.w;
            }
        }
#pragma unroll
        for (int j = 0; j < G; j++) r[j] = WIDE ? w[WIDE ? j : 0] : j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu;
        return any != 0;
    }
};

// The biases of a block's tokens among up to T entries of a row's list, in any order: the place in the list and the token in one word.
template <int T>
struct BiasList {
    uint32_t key[T];  // place << 16 | token, from the block's first on
    float value[T];
    uint32_t named[(T == 512 ? kRuleSpan : kRuleWhole) / 32];  // a bit per token: whether there is an entry
    int n, twice;  // entries; whether a token has two
    // v with the token's biases, in their order
    __device__ __forceinline__ float add(float v, uint32_t t) const {
        uint32_t from = 0;
        while (true) {
            uint32_t least = 0xFFFFFFFFu;
            float value_ = 0.f;
            for (int e = 0; e < n; e++)
                if ((key[e] & 0xFFFFu) == t && key[e] >= from && key[e] < least) {
                    least = key[e];
                    value_ = value[e];
                }
            if (least == 0xFFFFFFFFu) return v;
            v = __fadd_rn(v, value_);
            from = least + 1;
        }
    }
};

// DT: x's type. HIST: with counters. G: neighbouring logits of a thread. VEC: a row of x and the same one of out begin at the same place within groups of eight;
// the blocks' parts begin on groups, the first one's `shift` before the row. Rows of an odd vocabulary are taken in groups like this
// (eight rows of 151,665 4.0 us on one logit at a time, of 151,936 2.5).
template <int T, int G, int DT, bool HIST, bool WIDE, bool VEC>
__global__ void __launch_bounds__(T, T == 512 ? kRulePerSm : 1) logit_rules_kernel(const __grid_constant__ RuleParams p) {
    typedef Counter<WIDE> Count;
    typedef typename std::conditional<DT == kF32, float, uint16_t>::type E;
    extern __shared__ uint4 smem[];
    __shared__ BiasList<T> list;
    uint32_t* const count = reinterpret_cast<uint32_t*>(smem);
    const int tid = threadIdx.x;
    const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts;
    const int shift = VEC ? (int)((p.misplaced + (uint32_t)row * (uint32_t)(p.ldx & 7)) & (uint32_t)(G - 1)) : 0;
    const int lo = part * p.span - shift, n = max(min(p.span, p.vocab - lo), 0);  // this block's logits are lo .. lo + n, from 0 on
    pdl_launch_dependents();
    if (HIST)
        for (int i = tid; i < p.span / (WIDE ? 4 : 8); i += T) smem[i] = make_uint4(0, 0, 0, 0);
    if (p.r.bias_offsets != nullptr)
        for (int i = tid; i < p.span / 32; i += T) list.named[i] = 0;
    if (tid == 0) list.n = list.twice = 0;
    pdl_wait();
    const E* const x = static_cast<const E*>(p.x) + (size_t)row * p.ldx + lo;  // (of the block's logits)
    float* const out = p.out + (size_t)row * p.ldo + lo;
    auto load1 = [&](int i) {
        if (DT == kF32) return reinterpret_cast<const float*>(x)[i];
        const uint16_t h = reinterpret_cast<const uint16_t*>(x)[i];
        return DT == kBF16 ? bf16_bits_to_f32(h) : __half2float(__ushort_as_half(h));
    };
    // A thread has the groups tid, tid + T, ... of the part: those that lie in the row as a whole are turns first_ .. last_, one at
    // either end may not (the row's first and last logits).
    constexpr int kStep = G * T, kWords = DT == kF32 ? G : G / 2;
    constexpr int kBatch = DT == kF32 && G == 8 ? 1 : 2;  // groups of a thread that are under way at once
    const int first_ = lo + G * tid < 0 ? 1 : 0, last_ = n >= G * tid + G ? (n - G * tid - G) / kStep + 1 : 0;
    struct Group {
        uint32_t v[kWords];
    };
    auto load = [&](int turn) {
        const E* const q = x + G * tid + turn * kStep;
        Group f;
        if (VEC) {
            if (kWords == 8) {
                asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                             : "=r"(f.v[0]), "=r"(f.v[1]), "=r"(f.v[kWords == 8 ? 2 : 0]), "=r"(f.v[kWords == 8 ? 3 : 0]), "=r"(f.v[kWords == 8 ? 4 : 0]),
                               "=r"(f.v[kWords == 8 ? 5 : 0]), "=r"(f.v[kWords == 8 ? 6 : 0]), "=r"(f.v[kWords == 8 ? 7 : 0])
                             : "l"(q)
                             : "memory");
            } else if (kWords == 4) {
                const uint4 w = *reinterpret_cast<const uint4*>(q);
                f.v[0] = w.x; f.v[1] = w.y; f.v[kWords == 4 ? 2 : 0] = w.z; f.v[kWords == 4 ? 3 : 0] = w.w;
            } else {
                const uint2 w = *reinterpret_cast<const uint2*>(q);
                f.v[0] = w.x; f.v[1] = w.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < kWords; j++) {
                if (DT == kF32) f.v[j] = reinterpret_cast<const uint32_t*>(q)[j];
                else f.v[j] = (uint32_t)q[2 * j] | (uint32_t)q[2 * j + 1] << 16;
            }
        }
        return f;
    };
    // Everything that does not wait for something else first: the first logits, the row's numbers, the first tokens of its history
    Group ahead[kBatch] = {};
#pragma unroll
    for (int k = 0; k < kBatch; k++)
        if (first_ + k < last_) ahead[k] = load(first_ + k);
    const int32_t* const tokens = HIST ? p.r.tokens + (size_t)row * p.r.ld_tokens : nullptr;
    uint32_t look[kRuleLook];
    if (HIST) {
#pragma unroll
        for (int k = 0; k < kRuleLook; k++) look[k] = k * T + tid < p.r.max_tokens ? (uint32_t)tokens[k * T + tid] : 0xFFFFFFFFu;
    }
    const float rep = p.r.repetition != nullptr ? p.r.repetition[row] : 1.f, pres = p.r.presence != nullptr ? p.r.presence[row] : 0.f;
    const float freq = p.r.frequency != nullptr ? p.r.frequency[row] : 0.f;
    const int len = HIST ? min(max(p.r.lens[row], 0), p.r.max_tokens) : 0, said = HIST && p.r.prompt_lens != nullptr ? p.r.prompt_lens[row] : 0;
    const int m = p.r.mask == nullptr ? -1 : p.r.mask_rows != nullptr ? p.r.mask_rows[row] : row;
    const bool biases = p.r.bias_offsets != nullptr;
    // (cut to the list on both sides before anything is added to them)
    const int b0 = biases ? min(max(p.r.bias_offsets[row], 0), p.r.biases) : 0, b1 = biases ? max(min(p.r.bias_offsets[row + 1], p.r.biases), b0) : 0;
    __syncthreads();  // the counters are zero
    // the thread's entry of the row's biases from j0 on into the list; where it went, or -1
    auto collect = [&](int j0) {
        if (tid >= b1 - j0) return -1;
        const int j = j0 + tid;
        const uint32_t token = (uint32_t)p.r.bias_tokens[j], t = token - (uint32_t)lo;
        if (token >= (uint32_t)p.vocab || t >= (uint32_t)n) return -1;
        if (atomicOr(&list.named[t >> 5], 1u << (t & 31)) >> (t & 31) & 1) list.twice = 1;
        const int at = atomicAdd(&list.n, 1);
        list.key[at] = (uint32_t)tid << 16 | t;
        list.value[at] = p.r.bias_values[j];
        return at;
    };
    // A token's biases are in the hands of the thread that has the first of them. Its logit is read before anything is written
    // (x may be out) and its result stored behind all the others.
    const int mine = b0 < b1 ? collect(b0) : -1;
    const uint32_t my_token = mine >= 0 ? list.key[mine] & 0xFFFFu : 0;
    const float my_logit = mine >= 0 ? load1(my_token) : 0.f;
    const uint32_t* const mask = m >= 0 && m < p.r.masks ? p.r.mask + (size_t)m * p.r.ld_mask : nullptr;
    // the bits of a whole group: a turn is whole words on, and the place in a word stays
    const int mask_at = (lo + G * tid) & 31;
    const uint32_t* const mask_word = mask + ((lo + G * tid) >> 5);
    auto allowed = [&](int turn) {
        const uint32_t* const q = mask_word + turn * (kStep / 32);
        uint32_t bits = q[0] >> mask_at;
        if (VEC && mask_at > 32 - G) bits |= q[1] << (32 - mask_at);
        return bits;
    };
    uint32_t bits[kBatch] = {};
    if (mask != nullptr) {
#pragma unroll
        for (int k = 0; k < kBatch; k++)
            if (first_ + k < last_) bits[k] = allowed(first_ + k);
    }
    const bool counts = HIST && len > 0 && (rep != 1.f || pres != 0.f || freq != 0.f);
    if (counts) {
        const int prompt = min(max(said, 0), len);
        auto note = [&](int i, uint32_t token) {
            const uint32_t t = token - (uint32_t)lo;  // (-1 to -7 may find the places before the row, which nobody stores)
            if (i < len && t < (uint32_t)n) Count::note(count, t, i < prompt);
        };
#pragma unroll
        for (int k = 0; k < kRuleLook; k++) note(k * T + tid, look[k]);
        // Long histories by 4096 tokens that are all of the prompt or all generated (a load of 32 costs some ten instructions then, else thirty: the blocks of a
        // row all look at all of them)
        const bool whole = (reinterpret_cast<uintptr_t>(tokens) & 15) == 0;
        const uint32_t counters = smem_u32(count);
        for (int i0 = kRuleLook * T; i0 < len; i0 += 8 * T) {
            const int i1 = i0 + 8 * T;
            if (whole && i1 <= len && (i0 >= prompt || i1 <= prompt)) {
                const int4* const q = reinterpret_cast<const int4*>(tokens + i0) + tid;
                const int4 a = q[0], b = q[T];
                const uint32_t t[8] = {(uint32_t)a.x, (uint32_t)a.y, (uint32_t)a.z, (uint32_t)a.w, (uint32_t)b.x, (uint32_t)b.y, (uint32_t)b.z, (uint32_t)b.w};
                if (i0 >= prompt) {
#pragma unroll
                    for (int k = 0; k < 8; k++) Count::template note_if<false>(counters, t[k] - (uint32_t)lo, (uint32_t)n);
                } else {
#pragma unroll
                    for (int k = 0; k < 8; k++) Count::template note_if<true>(counters, t[k] - (uint32_t)lo, (uint32_t)n);
                }
                continue;
            }
            uint32_t t[8];
#pragma unroll
            for (int k = 0; k < 8; k++) t[k] = i0 + k * T + tid < len ? (uint32_t)tokens[i0 + k * T + tid] : 0xFFFFFFFFu;
#pragma unroll
            for (int k = 0; k < 8; k++) note(i0 + k * T + tid, t[k]);
        }
    }
    __syncthreads();  // every token is counted, every bias in the list

    auto one = [&](float l, uint32_t c) {
        if (c == 0) return l;
        l = l > 0.f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
        const uint32_t times = c & ~Count::PROMPT;
        l = __fsub_rn(l, __fmul_rn(freq, (float)times));
        return times != 0 ? __fsub_rn(l, pres) : l;
    };
    // a list's entry: whether no earlier one is of its token, and whether it is the only one
    auto first = [&](int at, bool& only) {
        const uint32_t key = list.key[at];
        bool yes = true;
        only = true;
        for (int e = 0; e < list.n; e++) {
            const bool same = (list.key[e] & 0xFFFFu) == (key & 0xFFFFu);
            yes = yes && (!same || list.key[e] >= key);
            only = only && (!same || e == at);
        }
        return yes;
    };
    auto may1 = [&](uint32_t t) { return mask == nullptr || (mask[(lo + (int)t) >> 5] >> ((lo + (int)t) & 31) & 1); };
    float my_result = 0.f;
    bool store = false;
    if (mine >= 0) {
        bool only = true;
        store = list.twice == 0 || first(mine, only);  // (a look at the whole list only where it has to be)
        if (store) {
            my_result = HIST && counts ? one(my_logit, Count::one(count, my_token)) : my_logit;
            my_result = only ? __fadd_rn(my_result, list.value[mine]) : list.add(my_result, my_token);
            if (!may1(my_token)) my_result = -INFINITY;
        }
    }
    auto finish = [&](int turn, const Group& f, uint32_t may) {
        const int i = G * tid + turn * kStep;
        float v[G];
        if (DT == kF32) {
#pragma unroll
            for (int j = 0; j < G; j++) v[j] = __uint_as_float(f.v[DT == kF32 ? j : 0]);
        } else {
#pragma unroll
            for (int j = 0; j < G / 2; j++) {
                if (DT == kBF16) {
                    v[2 * j] = __uint_as_float(f.v[j] << 16);
                    v[2 * j + 1] = __uint_as_float(f.v[j] & 0xFFFF0000u);
                } else {
                    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&f.v[j]));
                    v[2 * j] = a.x;
                    v[2 * j + 1] = a.y;
                }
            }
        }
        if (HIST && counts) {
            uint32_t c[G];
            if (Count::template group<G>(count, i, c)) {
#pragma unroll
                for (int j = 0; j < G; j++) v[j] = one(v[j], c[j]);
            }
        }
        if (mask != nullptr) {
#pragma unroll
            for (int j = 0; j < G; j++)
                if (!(may >> j & 1)) v[j] = -INFINITY;
        }
        if (VEC) {
            if (G == 8)  // (a whole sector)
                asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(out + i), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[G - 4]),
                             "f"(v[G - 3]), "f"(v[G - 2]), "f"(v[G - 1])
                             : "memory");
            else *reinterpret_cast<float4*>(out + i) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int j = 0; j < G; j++) out[i + j] = v[j];
        }
    };
    for (int turn = first_; turn < last_; turn += kBatch) {
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            const Group f = ahead[k];
            const uint32_t may = bits[k];
            if (turn + k + kBatch < last_) {
                ahead[k] = load(turn + k + kBatch);
                if (mask != nullptr) bits[k] = allowed(turn + k + kBatch);
            }
            if (turn + k < last_) finish(turn + k, f, may);
        }
    }
    auto single = [&](int i) {
        if (i >= n || lo + i < 0) return;
        float v = load1(i);
        if (HIST && counts) v = one(v, Count::one(count, i));
        out[i] = may1(i) ? v : -INFINITY;
    };
    if (first_ == 1)
        for (int j = 0; j < G; j++) single(G * tid + j);
    const int end = G * tid + last_ * kStep;
    if (last_ >= first_ && end < n)
        for (int j = 0; j < G; j++) single(end + j);
    if (b0 < b1) {
        __syncthreads();
        if (store) out[my_token] = my_result;
    }
    // more biases than the list takes at once: by rounds
    for (int left = b1 - b0 - T; left > 0; left -= T) {
        __syncthreads();
        for (int i = tid; i < p.span / 32; i += T) list.named[i] = 0;
        if (tid == 0) list.n = list.twice = 0;
        __syncthreads();
        const int at = collect(b1 - left);
        __syncthreads();
        if (at >= 0) {
            const uint32_t t = list.key[at] & 0xFFFFu;
            bool only = true;
            if ((list.twice == 0 || first(at, only)) && may1(t)) out[t] = only ? __fadd_rn(out[t], list.value[at]) : list.add(out[t], t);
        }
    }
}

typedef void (*RulesKernel)(RuleParams);
enum { kNoHistory, kNarrow, kWide, kWhole };  // no counters; two of 16 bits in a word; of 32 bits; those and an SM to itself
template <int DT, bool VEC>
RulesKernel rules_pick(int kind, bool eight) {
    return kind == kNarrow  ? logit_rules_kernel<512, 4, DT, true, false, VEC>
           : kind == kWide  ? logit_rules_kernel<512, 4, DT, true, true, VEC>
           : kind == kWhole ? eight ? logit_rules_kernel<1024, 8, DT, true, true, VEC> : logit_rules_kernel<1024, 4, DT, true, true, VEC>
           : eight          ? logit_rules_kernel<512, 8, DT, false, false, VEC> : logit_rules_kernel<512, 4, DT, false, false, VEC>;
}
template <int DT>
RulesKernel rules_pick(int kind, bool eight, bool vec) { return vec ? rules_pick<DT, true>(kind, eight) : rules_pick<DT, false>(kind, eight); }
RulesKernel rules_pick(int dtype, int kind, bool eight, bool vec) {
    return dtype == kF32 ? rules_pick<kF32>(kind, eight, vec) : dtype == kF16 ? rules_pick<kF16>(kind, eight, vec) : rules_pick<kBF16>(kind, eight, vec);
}

}  // namespace

int32_t rules_init(iq_ctx* ctx) {
    for (int dtype = 0; dtype < 3; dtype++)
        for (int v = 0; v < 12; v++) {
            const int kind = kNarrow + v / 4;
            const cudaError_t e = cudaFuncSetAttribute(reinterpret_cast<const void*>(rules_pick(dtype, kind, (v & 2) != 0, (v & 1) != 0)), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       kind == kNarrow ? kRuleSpan * 2 : kind == kWide ? kRuleSpan * 4 : kRuleWhole * 4);
            if (e != cudaSuccess) return check_cuda(ctx, e, "cudaFuncSetAttribute(logit_rules)");
        }
    return kOk;
}

}  // namespace iq

using namespace iq;

extern "C" int32_t iq_logits_rules(iq_ctx* ctx, void* stream, const void* x, int32_t x_dtype, int64_t ldx, float* out, int64_t ldo, int32_t rows, int32_t vocab,
                                   const iq_logit_rules* rules) {
    // (the checks come before the context is looked at: they are the same without a GPU)
    if (x == nullptr || out == nullptr || rules == nullptr || x_dtype < 0 || x_dtype > 2) return fail(ctx, kErrInvalidArg, "logits_rules: null pointer, or x is not of fp32, fp16 or bf16");
    if (rows < 0 || vocab < 1 || ldx < vocab || ldo < vocab) return fail(ctx, kErrInvalidArg, "logits_rules: rows = %d, vocab = %d, rows at least vocab apart", rows, vocab);
    const iq_logit_rules& r = *rules;
    const int esz = dtype_size(x_dtype);
    uintptr_t words = reinterpret_cast<uintptr_t>(out);
    for (const void* t : {(const void*)r.tokens, (const void*)r.lens, (const void*)r.prompt_lens, (const void*)r.repetition, (const void*)r.presence, (const void*)r.frequency,
                          (const void*)r.bias_offsets, (const void*)r.bias_tokens, (const void*)r.bias_values, (const void*)r.mask, (const void*)r.mask_rows})
        words |= reinterpret_cast<uintptr_t>(t);
    if (words % 4 != 0 || reinterpret_cast<uintptr_t>(x) % esz != 0) return fail(ctx, kErrInvalidArg, "logits_rules: a tensor does not begin on an element");
    if (vocab > kRuleMaxVocab || rows > (1 << 24)) return fail(ctx, kErrUnsupported, "logits_rules: rows = %d, vocab = %d (up to %d rows of %d logits)", rows, vocab, 1 << 24, kRuleMaxVocab);
    if (r.tokens != nullptr && (r.lens == nullptr || r.max_tokens < 0 || r.ld_tokens < r.max_tokens))
        return fail(ctx, kErrInvalidArg, "logits_rules: a history has lengths, its rows at least max_tokens apart");
    if (r.tokens != nullptr && r.max_tokens > kRuleMaxTokens) return fail(ctx, kErrUnsupported, "logits_rules: a history of up to %d tokens", kRuleMaxTokens);
    if (r.bias_offsets != nullptr && (r.biases < 0 || (r.biases > 0 && (r.bias_tokens == nullptr || r.bias_values == nullptr))))
        return fail(ctx, kErrInvalidArg, "logits_rules: biases are offsets, tokens and values");
    if (r.mask != nullptr && (r.masks < 1 || r.ld_mask < (vocab + 31) / 32 || (r.mask_rows == nullptr && r.masks < rows)))
        return fail(ctx, kErrInvalidArg, "logits_rules: a mask per row or mask_rows, of at least %d words", (vocab + 31) / 32);
    if (ctx == nullptr) return kErrInvalidArg;
    if (rows == 0) return kOk;
    RuleParams p;
    p.x = x; p.ldx = ldx; p.out = out; p.ldo = ldo; p.vocab = vocab; p.r = r;
    const bool hist = r.tokens != nullptr && r.max_tokens > 0 && (r.repetition != nullptr || r.presence != nullptr || r.frequency != nullptr);
    int kind = !hist ? kNoHistory : r.max_tokens > 0x7FFF ? kWide : kNarrow;
    // Logits of a block where the rows have so many blocks. With a history and where that fits, a block of 1024 threads per SM: every block looks at the whole
    // list, and counters of 32 bits take half the instructions. Otherwise three of 512 per SM, in whole rounds, as few as the largest span allows: their phases
    // overlap (without a history 64 rows of 262,144 22.6 us). Of blocks with 32-bit counters for more than some 17,000 logits only two fit, and the rounds are not
    // whole: a capacity of 131,072 tokens instead of 16,384, 2048 of them used, takes 64 rows of 262,144 in bf16 from 22.5 to 27.0 us, 256 of 128,000 from 42.8 to 51.8. One / three blocks per SM, 16,384 (500) tokens, us: one row of 128,000 4.1 / 5.0 (2.4 / 2.3),
    // 8 of 151,665 6.6 / 9.2 (3.9 / 4.3), 64 of 32,000 8.6 / 12.2 (4.4 / 5.4), 24 of 151,665 11.6 / 14.9 (8.0 / 7.9), with 50,555 logits per block 40 of
    // 151,665 16.8 / 17.9 (13.4 / 10.9).
    auto span = [&](int64_t blocks, int least) {
        const int64_t parts = std::max<int64_t>(blocks / rows, 1);
        return std::max((int)((vocab + 7 + parts - 1) / parts + 127) / 128 * 128, least);
    };
    if (hist && rows <= ctx->sms && span(ctx->sms, kRuleLeast / 2) <= kRuleWhole) {
        kind = kWhole;
        p.span = span(ctx->sms, kRuleLeast / 2);
    } else {
        for (int64_t rounds = 1; rounds == 1 || p.span > kRuleSpan; rounds++) p.span = span(kRulePerSm * ctx->sms * rounds, kRuleLeast);
    }
    p.parts = (vocab + 7 + p.span - 1) / p.span;  // (a row may begin seven elements into the first one's)
    p.misplaced = (uint32_t)(reinterpret_cast<uintptr_t>(x) / esz & 7);
    const bool vec = (reinterpret_cast<uintptr_t>(out) / 4 & 7) == p.misplaced && ((ldx ^ ldo) & 7) == 0;
    // Groups of eight logits from one and a half turns of the threads on, where the registers hold them: 64 rows of 262,144 in bf16 without a history 19.0 -> 17.3 us,
    // under grammars 22.0 -> 18.7, 16 of 128,000 with 2048 tokens 5.4 -> 4.9; but 8 of 151,665 (8448 logits per block) 4.8 -> 5.5.
    const bool eight = p.span >= 12 * (kind == kWhole ? 1024 : 512);
    const RulesKernel kernel = rules_pick(x_dtype, kind, eight, vec);
    DeviceScope on(ctx);
    if (on.error != cudaSuccess) return check_cuda(ctx, on.error, "logits_rules device");
    return check_cuda(ctx, launch_dependent(kernel, dim3((unsigned)rows * p.parts), kind == kWhole ? 1024 : 512, hist ? (size_t)p.span * (kind == kNarrow ? 2 : 4) : 0, reinterpret_cast<cudaStream_t>(stream), p),
                      "logits_rules launch");
}
