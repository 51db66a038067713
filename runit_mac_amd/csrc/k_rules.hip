// k_rules.hip — rules on logits: penalties for repeated tokens, biases, grammar
// masks.
//
// Of a token that its row's list has c times, c' of them behind the prompt, and
// whose biases sum to b:
//   x → (c > 0: x > 0 ? x / rep : x·rep) − freq·c' − (c' > 0 ? pres : 0) + b,
// −∞ where the row's mask has no bit for it; in f32, rounded once.
//
// A workgroup has RT_RULES_SEG tokens of a row.  It counts the list's tokens
// among them in LDS (whole numbers: any order), and sums their biases there in the
// list's order, each by the thread whose entry is the token's first.  In place only
// the logits that change are written, and only those that no mask forbids
// read.  Bound by the logits' bytes; few rows: by trips to memory.
#include "rt_attn.h"

template <class T>
struct RuleVec;
template <>
struct RuleVec<float> {
    static constexpr uint32_t N = 4;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct RuleVec<_Float16> {
    static constexpr uint32_t N = 8;
    typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
};

template <class T>
RT_DEV void adjust_logits(const RulesArgs& a) {
    constexpr uint32_t SEG = RT_RULES_SEG, N = RuleVec<T>::N;
    constexpr uint32_t PROMPT = 0x80000000u;  // in the prompt; the other bits count behind it
    typedef typename RuleVec<T>::vec vec;
    __shared__ uint32_t count[SEG];
    __shared__ float more[SEG];
    __shared__ uint32_t twice;
    const uint32_t tid = threadIdx.x, row = blockIdx.y, e0 = blockIdx.x * SEG, e1 = min(a.n, e0 + SEG);
    const T* x = (const T*)a.x + row * a.row_stride;
    T* out = (T*)a.out + row * a.row_stride;
    auto list = [&](const uint32_t* start, const uint32_t* len, uint64_t n, uint64_t& at) {
        at = start[row];
        return at < n ? (uint32_t)min((uint64_t)len[row], n - at) : 0u;
    };
    uint64_t ta = 0, ba = 0;
    const uint32_t nt = a.tokens ? list(a.token_start, a.token_len, a.n_tokens, ta) : 0;
    const uint32_t nb = a.bias_ids ? list(a.bias_start, a.bias_len, a.n_bias, ba) : 0;
    const uint32_t np = a.prompt_len && nt ? a.prompt_len[row] : 0;
    const float rep = a.repetition && nt ? a.repetition[row] : 1.0f, freq = a.frequency && nt ? a.frequency[row] : 0.0f,
                pres = a.presence && nt ? a.presence[row] : 0.0f;
    const uint32_t mr = !a.mask ? 0xffffffffu : a.mask_row ? a.mask_row[row] : row;
    const uint32_t* mask = mr < a.mask_rows ? a.mask + mr * a.mask_stride : nullptr;
    if (nb) {
        const uint32_t* ids = a.bias_ids + ba;
        for (uint32_t i = tid; i < SEG; i += 256) count[i] = 0xffffffffu, more[i] = 0.0f;
        if (tid == 0) twice = 0;
        __syncthreads();
        for (uint32_t j = tid; j < nb; j += 256)
            if (ids[j] - e0 < e1 - e0) atomicMin(&count[ids[j] - e0], j);
        __syncthreads();
        for (uint32_t j = tid; j < nb; j += 256)
            if (ids[j] - e0 < e1 - e0 && count[ids[j] - e0] != j) twice = 1;
        __syncthreads();
        const bool again = twice;
        for (uint32_t j = tid; j < nb; j += 256) {
            const uint32_t k = ids[j] - e0;
            if (k >= e1 - e0 || count[k] != j) continue;
            float s = a.bias[ba + j];
            for (uint32_t i = j + 1; again && i < nb; ++i)
                if (ids[i] == ids[j]) s += a.bias[ba + i];
            more[k] = s;
        }
        __syncthreads();
    }
    if (nt) {
        for (uint32_t i = tid; i < SEG; i += 256) count[i] = 0;
        __syncthreads();
        for (uint32_t j = tid; j < nt; j += 256) {
            const uint32_t k = a.tokens[ta + j] - e0;
            if (k >= e1 - e0) continue;
            if (j < np) atomicOr(&count[k], PROMPT);
            else atomicAdd(&count[k], 1u);
        }
        __syncthreads();
    }
    for (uint32_t i = e0 + tid * N; i < e1; i += 256 * N) {
        const uint32_t m = min(N, e1 - i);
        uint32_t ok = (1u << N) - 1;
        if (mask) ok &= mask[i / 32] >> i % 32;  // (N divides 32, and e0 by it)
        uint32_t c[N], some = 0;
        float b[N];
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            c[k] = nt ? count[i - e0 + k] : 0;
            b[k] = nb ? more[i - e0 + k] : 0.0f;
            some |= c[k] || b[k] != 0.0f ? 1u << k : 0;
        }
        some &= ok;
        T v[N];
        if (!a.inplace || some) {
            if (m == N) {
                const vec y = *(const vec*)(x + i);
#pragma unroll
                for (uint32_t k = 0; k < N; ++k) v[k] = y[k];
            } else {
                for (uint32_t k = 0; k < N; ++k) v[k] = k < m ? x[i + k] : (T)0;
            }
        }
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            if (some >> k & 1) {
                float y = (float)v[k];
                const uint32_t said = c[k] & ~PROMPT;
                if (c[k]) y = y > 0.0f ? y / rep : y * rep;
                if (said) y = y - freq * (float)said - pres;
                v[k] = (T)(y + b[k]);
            }
            if (!(ok >> k & 1)) v[k] = (T)-__builtin_huge_valf();
        }
        const uint32_t all = (1u << N) - 1, write = a.inplace ? some | (all & ~ok) : all;
        if (write == all && m == N) {
            vec y;
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) y[k] = v[k];
            *(vec*)(out + i) = y;
        } else {
            for (uint32_t k = 0; k < N; ++k)
                if (k < m && write >> k & 1) out[i + k] = v[k];
        }
    }
}
extern "C" __global__ void __launch_bounds__(256) k_adjust_logits_f32(RulesArgs a) { adjust_logits<float>(a); }
extern "C" __global__ void __launch_bounds__(256) k_adjust_logits_f16(RulesArgs a) { adjust_logits<_Float16>(a); }
