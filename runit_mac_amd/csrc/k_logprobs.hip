// k_logprobs.hip — the log probability of a given token per row of logits,
// with the row's entropy, the token's rank and the most probable tokens.
//
// One pass over the logits: with m the running maximum, S = Σ e^(x−m) and
// U = Σ e^(x−m)·(m − x),
//   log p(t) = x_t − m − ln S,   entropy = ln S + U / S
// (U from the distances to the maximum, so that a confident row's small entropy
// is no difference of large numbers).  A thread keeps m, S and U of its own
// elements and rescales when its maximum grows.
//
// The largest `top` values: each wave keeps them sorted, one a lane, as 64-bit
// keys (the float's order above the complement of its index: equal values go by
// the lower index), and inserts the few that beat the last.
#include "rt_attn.h"

typedef unsigned long long u64_t;

// the order of the floats as whole numbers, −∞ and NaN below all others, both zeros alike
RT_DEV uint32_t float_order(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return x != x ? 0x007fffffu : b >> 31 ? ~b : b | 0x80000000u;
}
RT_DEV float order_float(uint32_t k) {
    return __builtin_bit_cast(float, k >> 31 ? k & 0x7fffffffu : ~k);
}
RT_DEV u64_t shfl64(u64_t v, int l) { return __shfl(v, l, 64); }

// A wave's sorted list (lane i: the i-th largest key; 0: none).
struct TopList {
    u64_t key = 0, last = 0;  // last: the key that a new one has to beat
    RT_DEV void insert(u64_t k, uint32_t top) {  // k: the same in every lane
        const uint32_t lane = threadIdx.x & 63, at = __popcll(__ballot(key > k));
        const u64_t up = __shfl_up(key, 1, 64);
        key = lane < at ? key : lane == at ? k : up;
        last = shfl64(key, top - 1);
    }
    // one key of each lane
    RT_DEV void offer(u64_t k, uint32_t top) {
        u64_t hit = __ballot(k > last);
        while (hit) {
            const int l = __builtin_ctzll(hit);
            const u64_t x = shfl64(k, l);
            if (x > last) insert(x, top);
            hit &= hit - 1;
        }
    }
};

struct LogSum {
    float m = -__builtin_huge_valf(), s = 0.0f, u = 0.0f;
    // the sums measured from another maximum (≥ m)
    RT_DEV void to(float m2) {
        const float d = m2 - m, f = m == -__builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(-d * 1.44269504f);
        u = f > 0.0f ? f * fmaf(d, s, u) : f * u;  // (f = 0: no 0·∞)
        s *= f;
        m = m2;
    }
    RT_DEV void add(float x) {  // x ≤ m, or NaN
        const float md = m == -__builtin_huge_valf() ? 0.0f : m, d = md - x;
        const float e = __builtin_amdgcn_exp2f(-d * 1.44269504f);
        s += e;
        u += e > 0.0f ? e * d : 0.0f;
    }
    RT_DEV void join(float m2, float s2, float u2) {
        LogSum o;
        o.m = m2, o.s = s2, o.u = u2;
        const float M = fmaxf(m, m2);
        to(M);
        o.to(M);
        s += o.s;
        u += o.u;
    }
};

RT_DEV void logprobs_finish(const LogprobsArgs& a, uint32_t row, const LogSum& t, float xt, uint32_t rank,
                            u64_t key, bool scalar) {
    const uint32_t lane = threadIdx.x & 63;
    const float z = logf(t.s);
    if (scalar) {
        a.logprob[row] = xt - t.m - z;
        if (a.entropy) a.entropy[row] = z + t.u / t.s;
        if (a.rank) a.rank[row] = rank;
    }
    if (lane < a.top) {
        a.top_ids[(size_t)row * a.top + lane] = ~(uint32_t)key;
        a.top_logprobs[(size_t)row * a.top + lane] = order_float((uint32_t)(key >> 32)) - t.m - z;
    }
}

template <class T>
struct LogitVec;
template <>
struct LogitVec<float> {
    static constexpr uint32_t N = 4;
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct LogitVec<_Float16> {
    static constexpr uint32_t N = 8;
    typedef _Float16 vec __attribute__((ext_vector_type(8), aligned(2)));
};

// Grid (segments, rows), 4 waves.  A wave takes every fourth 64·N elements of
// its segment, so that its keys come in index order.
template <class T, bool TOP>
RT_DEV void logprobs(const LogprobsArgs& a) {
    constexpr uint32_t N = LogitVec<T>::N;
    __shared__ float red[4][3];
    __shared__ uint32_t ranks[4];
    __shared__ u64_t lists[4][64];
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t row = blockIdx.y, seg = blockIdx.x;
    const T* x = (const T*)a.x + row * a.row_stride;
    const uint32_t e0 = seg * a.seg_len, e1 = min(a.n, e0 + a.seg_len);
    const uint32_t tok = a.tokens[row];
    const float xt = tok < a.n ? (float)x[tok] : -__builtin_huge_valf();
    LogSum t;
    TopList best;
    uint32_t more = 0;
    for (uint32_t b = e0 + w * 64 * N; b < e1; b += 256 * N) {
        const uint32_t i = b + lane * N;
        float v[N];
        if (b + 64 * N <= e1) {
            const typename LogitVec<T>::vec r = *(const typename LogitVec<T>::vec*)(x + i);
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) v[k] = (float)r[k];
        } else {
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) v[k] = i + k < e1 ? (float)x[i + k] : -__builtin_huge_valf();
        }
        float mx = v[0];
#pragma unroll
        for (uint32_t k = 1; k < N; ++k) mx = fmaxf(mx, v[k]);
        if (mx > t.m) t.to(mx);
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            t.add(v[k]);
            more += v[k] > xt;
        }
        if constexpr (TOP) {
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) {
                const uint32_t id = i + k;
                best.offer(id < e1 ? (u64_t)float_order(v[k]) << 32 | (uint32_t)~id : 0, a.top);
            }
        }
    }
    for (int o = 32; o; o /= 2) {
        const float m2 = __shfl_xor(t.m, o, 64), s2 = __shfl_xor(t.s, o, 64), u2 = __shfl_xor(t.u, o, 64);
        t.join(m2, s2, u2);
        more += __shfl_xor(more, o, 64);
    }
    if (lane == 0) {
        red[w][0] = t.m, red[w][1] = t.s, red[w][2] = t.u;
        ranks[w] = more;
    }
    if constexpr (TOP) lists[w][lane] = best.key;
    __syncthreads();
    if (w) return;
    LogSum all;
    uint32_t rank = 0;
    for (uint32_t k = 0; k < 4; ++k) {
        all.join(red[k][0], red[k][1], red[k][2]);
        rank += ranks[k];
    }
    if constexpr (TOP)
        for (uint32_t k = 1; k < 4; ++k) best.offer(lane < a.top ? lists[k][lane] : 0, a.top);
    if (a.segs == 1) {
        logprobs_finish(a, row, all, xt, rank, best.key, lane == 0);
        return;
    }
    const size_t p = (size_t)row * a.segs + seg;
    if (lane == 0) {
        a.part[4 * p] = all.m, a.part[4 * p + 1] = all.s, a.part[4 * p + 2] = all.u;
        ((uint32_t*)a.part)[4 * p + 3] = rank;
    }
    if (lane < a.top) a.keys[p * a.top + lane] = best.key;
}

// One wave a row: a lane takes a segment's sums, and the lists one after another.
template <class T>
RT_DEV void logprobs_merge(const LogprobsArgs& a) {
    const uint32_t lane = threadIdx.x & 63, row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.row_stride;
    const uint32_t tok = a.tokens[row];
    const float xt = tok < a.n ? (float)x[tok] : -__builtin_huge_valf();
    LogSum t;
    uint32_t rank = 0;
    if (lane < a.segs) {
        const size_t p = (size_t)row * a.segs + lane;
        t.m = a.part[4 * p], t.s = a.part[4 * p + 1], t.u = a.part[4 * p + 2];
        rank = ((const uint32_t*)a.part)[4 * p + 3];
    }
    for (int o = 32; o; o /= 2) {
        const float m2 = __shfl_xor(t.m, o, 64), s2 = __shfl_xor(t.s, o, 64), u2 = __shfl_xor(t.u, o, 64);
        t.join(m2, s2, u2);
        rank += __shfl_xor(rank, o, 64);
    }
    TopList best;
    if (a.top)
        for (uint32_t s = 0; s < a.segs; ++s)
            best.offer(lane < a.top ? a.keys[((size_t)row * a.segs + s) * a.top + lane] : 0, a.top);
    logprobs_finish(a, row, t, xt, rank, best.key, lane == 0);
}

#define RT_LOGPROBS_KERNELS(S, T)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) k_logprobs_##S(LogprobsArgs a) { logprobs<T, false>(a); } \
    extern "C" __global__ void __launch_bounds__(256) k_logprobs_top_##S(LogprobsArgs a) { logprobs<T, true>(a); } \
    extern "C" __global__ void __launch_bounds__(64) k_logprobs_merge_##S(LogprobsArgs a) { logprobs_merge<T>(a); }
RT_LOGPROBS_KERNELS(f32, float)
RT_LOGPROBS_KERNELS(f16, _Float16)
