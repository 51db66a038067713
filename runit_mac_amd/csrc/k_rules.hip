// k_rules.hip — rules on logits: penalties for repeated tokens, biases, grammar
// masks.
//
// Of a token that its row's list has c times, c' of them behind the prompt, and
// whose biases sum to b:
//   x → (c > 0: x > 0 ? x / rep : x·rep) − freq·c' − (c' > 0 ? pres : 0) + b,
// −∞ where the row's mask has no bit for it; in f32, f16 logits rounded to f16 at the end.
//
// A workgroup has RT_RULES_SEG tokens of a row.  Its logits are on their way (where
// all are copied) while it counts the list's tokens among its own in LDS (whole
// numbers: any order) and puts their biases there.  Where two biases meet in
// a token it adds them again, one of a token a round, in the list's order.  In place only the
// logits that change are written, and only those that no mask forbids read.
//
// Bound by the logits' bytes: 120 rows of 152,064 f32 with histories of up to 9,000
// tokens, up to 300 biases and masks 33.7 µs for 147 MB (4.4 TB/s; a large copy makes
// 5.1; without lists 29).  Few rows: by trips to memory, 5 rows 4.1 µs, 4.4 a call.  4,096
// tokens and 512 threads: with 256 threads 39 µs, with 8,192 tokens 41, one thread
// adding all biases of its token one after another 68.
#include "rt_attn.h"

constexpr uint32_t NT = RT_RULES_THREADS;

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

// A list's entries, UNROLL of a thread at a time: those from j0 on into id, and f(entry, its place) of them.
template <uint32_t UNROLL>
RT_DEV void load_entries(const uint32_t* ids, uint32_t n, uint32_t j0, uint32_t (&id)[UNROLL]) {
#pragma unroll
    for (uint32_t u = 0; u < UNROLL; ++u) {
        const uint32_t j = j0 + NT * u + threadIdx.x;
        id[u] = j < n ? ids[j] : 0xffffffffu;
    }
}
template <uint32_t UNROLL, class F>
RT_DEV void each_entry(const uint32_t* ids, uint32_t n, uint32_t (&id)[UNROLL], const F& f) {
    for (uint32_t j0 = 0;;) {
#pragma unroll
        for (uint32_t u = 0; u < UNROLL; ++u) {
            const uint32_t j = j0 + NT * u + threadIdx.x;
            if (j < n) f(id[u], j);
        }
        if (n - j0 <= NT * UNROLL) break;
        j0 += NT * UNROLL;
        load_entries<UNROLL>(ids, n, j0, id);
    }
}

template <class T>
RT_DEV void adjust_logits(const RulesArgs& a) {
    constexpr uint32_t SEG = RT_RULES_SEG, N = RuleVec<T>::N, VECS = SEG / (NT * N);
    constexpr uint32_t PROMPT = 0x80000000u;  // in the prompt; the other bits count behind it
    typedef typename RuleVec<T>::vec vec;
    typedef uint32_t cvec __attribute__((ext_vector_type(4)));
    __shared__ cvec count4[SEG / 4];
    __shared__ f32x4 more4[SEG / 4];
    __shared__ uint32_t twice;
    uint32_t* count = (uint32_t*)count4;
    float* more = (float*)more4;
    const uint32_t tid = threadIdx.x, b0 = blockIdx.x, rest = b0 - a.rows, more_segs = a.segs - 1;
    // (all rows' first segments, then the rows': a text's commonest tokens have the lowest ids)
    const bool first = b0 < a.rows;
    // (the quotient from a product: below 2^24, off by one at most)
    uint32_t q = (uint32_t)((float)rest * a.inv_more);
    q -= q * more_segs > rest ? 1u : 0u;
    q += (q + 1) * more_segs <= rest ? 1u : 0u;
    const uint32_t row = __builtin_amdgcn_readfirstlane(first ? b0 : q);
    const uint32_t seg = __builtin_amdgcn_readfirstlane(first ? 0 : 1 + rest - q * more_segs);
    const uint32_t e0 = seg * SEG, e1 = min(a.n, e0 + SEG);
    const T* x = (const T*)a.x + row * a.row_stride;
    T* out = (T*)a.out + row * a.row_stride;
    vec v[VECS];  // (vector u: logits e0 + N·(threads·u + thread) ..; whole ones, where all are copied)
    if (!a.inplace) {
#pragma unroll
        for (uint32_t u = 0; u < VECS; ++u) {
            const uint32_t i = e0 + (NT * u + tid) * N;
            if (i + N <= e1) v[u] = *(const vec*)(x + i);
        }
    }
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
    uint32_t allowed[VECS];  // from the vector's first token on
#pragma unroll
    for (uint32_t u = 0; u < VECS; ++u) {
        const uint32_t i = e0 + (NT * u + tid) * N;
        allowed[u] = mr < a.mask_rows && i < e1 ? a.mask[mr * a.mask_stride + i / 32] >> i % 32 : 0xffffffffu;
    }
    if (nt || nb) {
        // (the lists' first entries are on their way while the counts are cleared)
        uint32_t said[8], biased[2];
        load_entries(a.tokens + ta, nt, 0, said);
        load_entries(a.bias_ids + ba, nb, 0, biased);
        for (uint32_t i = tid; i < SEG / 4; i += NT) {
            count4[i] = cvec{0, 0, 0, 0};
            more4[i] = f32x4{0, 0, 0, 0};
        }
        if (tid == 0) twice = 0;
        lds_barrier();
        each_entry(a.tokens + ta, nt, said, [&](uint32_t id, uint32_t j) {
            if (id - e0 >= e1 - e0) return;
            if (j < np) atomicOr(&count[id - e0], PROMPT);
            else atomicAdd(&count[id - e0], 1u);
        });
        // a bias alone is its token's; where two meet they are summed again, in order
        each_entry(a.bias_ids + ba, nb, biased, [&](uint32_t id, uint32_t j) {
            if (id - e0 >= e1 - e0) return;
            const uint32_t b = __builtin_bit_cast(uint32_t, a.bias[ba + j] + 0.0f);
            if (b && atomicExch((uint32_t*)&more[id - e0], b)) twice = 1;
        });
        lds_barrier();
        if (nb && twice) {
            // in rounds: of the entries of a token that are left the first is added (their places meet in the
            // counts' place, which wait in registers)
            constexpr uint32_t E = 4, NONE = 0xffffffffu;
            uint32_t kept[SEG / NT];
#pragma unroll
            for (uint32_t u = 0; u < SEG / NT; ++u) {
                kept[u] = count[NT * u + tid];
                count[NT * u + tid] = NONE;
                more[NT * u + tid] = 0.0f;
            }
            for (uint32_t j0 = 0; j0 < nb; j0 += NT * E) {
                uint32_t at[E];
                float b[E];
                bool left = false;
#pragma unroll
                for (uint32_t u = 0; u < E; ++u) {
                    const uint32_t j = j0 + NT * u + tid, k = j < nb ? a.bias_ids[ba + j] - e0 : NONE;
                    at[u] = k < e1 - e0 ? k : NONE;
                    b[u] = at[u] != NONE ? a.bias[ba + j] : 0.0f;
                    left |= at[u] != NONE;
                }
                while (__syncthreads_or(left)) {
#pragma unroll
                    for (uint32_t u = 0; u < E; ++u)
                        if (at[u] != NONE) atomicMin(&count[at[u]], NT * u + tid);
                    __syncthreads();
                    left = false;
#pragma unroll
                    for (uint32_t u = 0; u < E; ++u) {
                        if (at[u] == NONE) continue;
                        if (count[at[u]] == NT * u + tid) {
                            more[at[u]] += b[u];
                            count[at[u]] = NONE;  // (nobody else's place)
                            at[u] = NONE;
                        }
                        left |= at[u] != NONE;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (uint32_t u = 0; u < SEG / NT; ++u) count[NT * u + tid] = kept[u];
            __syncthreads();
        }
    }
    const bool lists = nt || nb;
#pragma unroll
    for (uint32_t u = 0; u < VECS; ++u) {
        const uint32_t i = e0 + (NT * u + tid) * N;
        if (i >= e1) break;
        const uint32_t m = min(N, e1 - i);
        const uint32_t ok = allowed[u] & ((1u << N) - 1);  // (N divides 32, and e0)
        uint32_t c[N], some = 0;
        float b[N];
        if (lists) {
#pragma unroll
            for (uint32_t k = 0; k < N; k += 4) {
                const cvec c4 = count4[(i - e0 + k) / 4];
                const f32x4 b4 = more4[(i - e0 + k) / 4];
#pragma unroll
                for (uint32_t w = 0; w < 4; ++w) {
                    c[k + w] = c4[w], b[k + w] = b4[w];
                    some |= c4[w] || b4[w] != 0.0f ? 1u << (k + w) : 0;
                }
            }
            some &= ok;
        }
        T y[N];
        if (!a.inplace && m == N) {
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) y[k] = v[u][k];
        } else if (!a.inplace || some) {
            for (uint32_t k = 0; k < N; ++k) y[k] = k < m ? x[i + k] : (T)0;
        }
        if (some) {
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) {
                if (!(some >> k & 1)) continue;
                float z = (float)y[k];
                const uint32_t said = c[k] & ~PROMPT;
                if (c[k]) z = z > 0.0f ? z / rep : z * rep;
                if (said) z = z - freq * (float)said - pres;
                y[k] = (T)(z + b[k]);
            }
        }
        const uint32_t all = (1u << N) - 1, write = a.inplace ? some | (all & ~ok) : all;
#pragma unroll
        for (uint32_t k = 0; k < N; ++k)
            if (!(ok >> k & 1)) y[k] = (T)-__builtin_huge_valf();
        if (write == all && m == N) {
            vec z;
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) z[k] = y[k];
            *(vec*)(out + i) = z;
        } else {
#pragma unroll
            for (uint32_t k = 0; k < N; ++k)
                if (k < m && write >> k & 1) out[i + k] = y[k];
        }
    }
}
extern "C" __global__ void __launch_bounds__(NT) k_adjust_logits_f32(RulesArgs a) { adjust_logits<float>(a); }
extern "C" __global__ void __launch_bounds__(NT) k_adjust_logits_f16(RulesArgs a) { adjust_logits<_Float16>(a); }
