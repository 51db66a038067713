// k_logprobs.hip — the log probability of a given token per row of logits,
// with the row's entropy, the token's rank and the most probable tokens.
//
// One pass over the logits: with m the running maximum, S = Σ e^(x−m) and
// U = Σ e^(x−m)·(m − x),
//   log p(t) = x_t − m − ln S,   entropy = ln S + U / S
// (U from the distances to the maximum, so that a confident row's small entropy
// is no difference of large numbers).  A thread keeps m, S and U of its own
// elements, in units of log 2, and rescales when its maximum grows.
//
// The largest `top` values: each wave keeps them sorted, one a lane, as 64-bit
// keys (the float's order above the complement of its index: equal values go by
// the lower index), and looks at a step's values one by one only if one of them
// reaches the smallest listed of any of the workgroup's waves; it gathers them
// in LDS and sorts them into the list many at a time (one by one as they came: 127
// µs for the first figure below).
//
// Bound by the logits' bytes, with many alternatives by the vector operations that
// look for them, with few rows by trips to memory: 500 rows of 152,064 f32 with
// 20 alternatives 74 µs, with 5 66, without 59 (304 MB, 5.2 TB/s; a large copy
// makes 5.1); 93 of 50,001 f16 without 8.4 (9.3 MB); 4 of 151,936 f32 with 5
// 11.6.  One workgroup of 16 waves a row instead of segments that meet was no
// faster from 93 rows on, and slower below.
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
template <uint32_t X>
RT_DEV u64_t lane_xor64(u64_t v) {
    return (u64_t)lane_xor<X>((uint32_t)(v >> 32)) << 32 | lane_xor<X>((uint32_t)v);
}
// the larger of lanes l and l ^ X in the lower of the two, whose bit B is clear
template <uint32_t X, uint32_t B>
RT_DEV u64_t order_lanes(u64_t k) {
    const u64_t o = lane_xor64<X>(k);
    return (o > k) != ((threadIdx.x & B) != 0) ? o : k;
}
// lane l's value (l the same in every lane), and that of the lane below (lane 0: 0), without LDS
RT_DEV u64_t lane64(u64_t v, uint32_t l) {
    return (u64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, l);
}
RT_DEV u64_t below64(u64_t v) {
    constexpr int WAVE_SHR_1 = 0x138;
    return (u64_t)(uint32_t)dpp_i<WAVE_SHR_1>((int)(v >> 32)) << 32 | (uint32_t)dpp_i<WAVE_SHR_1>((int)v);
}
// A wave's sorted list (lane i: the i-th largest key; 0: none).
struct TopList {
    u64_t key = 0, last = 0;  // last: the key that a new one has to beat
    RT_DEV void insert(u64_t k, uint32_t top) {  // k: the same in every lane
        const uint32_t lane = threadIdx.x & 63, at = __popcll(__ballot(key > k));
        const u64_t up = below64(key);
        key = lane < at ? key : lane == at ? k : up;
        last = lane64(key, top - 1);
    }
    // a falling sequence put behind a rising one, in falling order
    template <uint32_t D>
    static RT_DEV u64_t settle(u64_t k) {
        if constexpr (D > 0) return settle<D / 2>(order_lanes<D, D>(k));
        return k;
    }
    // the keys of the lanes in falling order: runs of S, each half's against the other's mirror
    template <uint32_t S = 2>
    static RT_DEV u64_t sort(u64_t k) {
        k = settle<S / 4>(order_lanes<S - 1, S / 2>(k));
        if constexpr (S < 64) return sort<S * 2>(k);
        return k;
    }
    // a sorted list of the same kind: the larger of its mirror and this one
    // holds the largest 64
    RT_DEV void merge(u64_t other, uint32_t top) {
        const u64_t o = lane_xor64<63>(other);
        key = settle<32>(key > o ? key : o);
        last = lane64(key, top - 1);
    }
    // one key of each lane, in any order
    RT_DEV void offer(u64_t k, uint32_t top) {
        u64_t hit = __ballot(k > last);
        if (__popcll(hit) > 12) {  // (that many insertions take as long as sorting them)
            merge(sort(k), top);
            return;
        }
        while (hit) {
            const u64_t x = lane64(k, __builtin_ctzll(hit));
            if (x > last) insert(x, top);
            hit &= hit - 1;
        }
    }
};

struct LogSum {
    float m = -__builtin_huge_valf(), s = 0.0f, u = 0.0f;  // m: of x; u in units of log 2, negative
    // the sums measured from another maximum (≥ m)
    RT_DEV void to(float m2) {
        const float d = (m - m2) * 1.44269504f, f = m == -__builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(d);
        u = f > 0.0f ? f * fmaf(d, s, u) : f * u;  // (f = 0: no 0·∞)
        s *= f;
        m = m2;
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
    RT_DEV void join_wave() {
        for (int o = 32; o; o /= 2) {
            const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64), u2 = __shfl_xor(u, o, 64);
            join(m2, s2, u2);
        }
    }
};

RT_DEV void logprobs_finish(const LogprobsArgs& a, uint32_t row, const LogSum& t, float xt, uint32_t rank,
                            u64_t key) {
    const uint32_t lane = threadIdx.x & 63;
    const float z = logf(t.s);
    if (lane == 0) {
        a.logprob[row] = xt - t.m - z;
        if (a.entropy) a.entropy[row] = z - 0.693147181f * (t.u / t.s);
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

// Grid (segments, rows), 4 waves.  A step is U vectors of N logits a thread,
// loaded while the one before is computed.  Rows in segments meet in the
// workgroup that arrives last.
template <class T, bool TOP>
RT_DEV void logprobs(const LogprobsArgs& a) {
    constexpr uint32_t N = LogitVec<T>::N, U = 16 / N, STEP = 256 * N * U;
    typedef typename LogitVec<T>::vec vec;
    __shared__ float red[4][3];
    __shared__ uint32_t ranks[4], floor_s, turn;
    constexpr uint32_t QUEUE = TOP ? 64 + 64 * N * U : 1;  // (below 64 are left by a step, it adds all at most)
    __shared__ u64_t lists[4][64], queue[4][QUEUE];
    const float NEG = -__builtin_huge_valf();
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const uint32_t row = blockIdx.y, seg = blockIdx.x;
    const T* x = (const T*)a.x + row * a.row_stride;
    const uint32_t e0 = seg * a.seg_len, e1 = min(a.n, e0 + a.seg_len);
    vec r[U];
    // vector u of a step at b: logits b + 256·N·u + N·thread ...; whole ones only
    auto load = [&](uint32_t b) {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t i = b + 256 * N * u + N * tid;
            if (i + N <= e1) r[u] = *(const vec*)(x + i);
        }
    };
    if (e0 < e1) load(e0);
    const uint32_t tok = a.tokens[row];
    const float xt = tok < a.n ? (float)x[tok] : NEG;
    const float xr = xt != xt ? NEG : xt;  // (NaN ranks as −∞)
    if (TOP && tid == 0) floor_s = 0;
    if constexpr (TOP) __syncthreads();
    LogSum t;
    TopList best;
    uint32_t more = 0, queued = 0;
    auto empty = [&]() {
        const u64_t was = best.last;
#pragma unroll 1
        for (uint32_t i = 0; i < queued; i += 64) best.offer(i + lane < queued ? queue[w][i + lane] : 0, a.top);
        if (best.last != was && lane == 0) atomicMax(&floor_s, (uint32_t)(best.last >> 32));
        queued = 0;
    };
    for (uint32_t b = e0; b < e1; b += STEP) {
        float v[U][N], mu[U], mx = NEG;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t i = b + 256 * N * u + N * tid;
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) v[u][k] = (float)r[u][k];
            if (i + N > e1) {
#pragma unroll
                for (uint32_t k = 0; k < N; ++k) v[u][k] = i + k < e1 ? (float)x[i + k] : NEG;
            }
            mu[u] = v[u][0];
#pragma unroll
            for (uint32_t k = 1; k < N; ++k) mu[u] = fmaxf(mu[u], v[u][k]);
            mx = fmaxf(mx, mu[u]);
        }
        if (b + STEP < e1) load(b + STEP);
        if (mx > t.m) t.to(mx);
        const float mm = t.m == NEG ? 0.0f : t.m;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u)
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) {
                // (the difference first: the type's lowest value times 1.44 is none)
                const float d = (v[u][k] - mm) * 1.44269504f, e = __builtin_amdgcn_exp2f(d);
                t.s += e;
                t.u = fmaf(e, fmaxf(d, -1e30f), t.u);  // (−∞: 0)
                more += v[u][k] > xr;
            }
        if constexpr (TOP) {
            uint32_t fl = *(volatile uint32_t*)&floor_s;
            // at first: as many of the lanes' maxima are no smaller than the top-th of them
            if (b == e0) fl = max(fl, (uint32_t)(lane64(TopList::sort((u64_t)float_order(mx) << 32), a.top - 1) >> 32));
            const float thr = order_float(fl);  // (NaN at 0)
            if (__ballot(!(mx < thr))) {
                // what reaches it into the wave's queue, from there into its list when
                // they are as many as it holds
#pragma unroll
                for (uint32_t u = 0; u < U; ++u) {
                    if (!__ballot(!(mu[u] < thr))) continue;
#pragma unroll
                    for (uint32_t k = 0; k < N; ++k) {
                        const uint32_t id = b + 256 * N * u + N * tid + k;
                        const bool in = id < e1 && !(v[u][k] < thr);
                        const uint64_t hit = __ballot(in);
                        if (hit) {
                            if (in)
                                queue[w][queued + __popcll(hit & ((1ull << lane) - 1))] =
                                    (u64_t)float_order(v[u][k]) << 32 | (uint32_t)~id;
                            queued += __popcll(hit);
                        }
                    }
                }
                if (queued >= min(64u, a.top) || b == e0) empty();
            }
        }
    }
    if constexpr (TOP) empty();
    t.join_wave();
    for (int o = 32; o; o /= 2) more += __shfl_xor(more, o, 64);
    if (lane == 0) {
        red[w][0] = t.m, red[w][1] = t.s, red[w][2] = t.u;
        ranks[w] = more;
    }
    // the four lists in two rounds
    auto meet = [&]() {
        if constexpr (TOP) {
            if (w & 1) lists[w][lane] = best.key;
            __syncthreads();
            if (!(w & 1)) best.merge(lists[w + 1][lane], a.top);
            if (w == 2) lists[w][lane] = best.key;
            __syncthreads();
            if (w == 0) best.merge(lists[2][lane], a.top);
        } else {
            __syncthreads();
        }
    };
    meet();
    LogSum all;
    uint32_t rank = 0;
    for (uint32_t k = 0; k < 4; ++k) {
        all.join(red[k][0], red[k][1], red[k][2]);
        rank += ranks[k];
    }
    if (a.segs == 1) {
        if (w == 0) logprobs_finish(a, row, all, xt, rank, best.key);
        return;
    }
    const size_t p = (size_t)row * a.segs;
    if (w == 0) {
        if (lane == 0) {
            dev_store(a.part + 2 * (p + seg), (uint64_t)__builtin_bit_cast(uint32_t, all.s) << 32 | __builtin_bit_cast(uint32_t, all.m));
            dev_store(a.part + 2 * (p + seg) + 1, (uint64_t)rank << 32 | __builtin_bit_cast(uint32_t, all.u));
        }
        if (TOP && lane < a.top) dev_store(a.keys + (p + seg) * a.top + lane, (uint64_t)best.key);
        dev_stores_done();
    }
    __syncthreads();
    if (tid == 0) {
        turn = arrive(a.counters + row);
        if (turn == a.segs - 1) dev_store(a.counters + row, 0u);
    }
    __syncthreads();
    if (turn != a.segs - 1) return;
    // all segments' sums, a lane each, and keys
    LogSum sum;
    uint32_t above = 0;
    if (lane < a.segs) {
        const uint64_t ms = dev_load(a.part + 2 * (p + lane)), ur = dev_load(a.part + 2 * (p + lane) + 1);
        sum.m = __builtin_bit_cast(float, (uint32_t)ms);
        sum.s = __builtin_bit_cast(float, (uint32_t)(ms >> 32));
        sum.u = __builtin_bit_cast(float, (uint32_t)ur);
        above = (uint32_t)(ur >> 32);
    }
    if constexpr (TOP) {
        best = TopList{};
        const uint32_t nk = a.segs * a.top;
        for (uint32_t k0 = 0; k0 < nk; k0 += 1024) {
            u64_t k[4];
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
                const uint32_t i = k0 + 256 * u + tid;
                k[u] = i < nk ? dev_load(a.keys + p * a.top + i) : 0;
            }
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) best.offer(k[u], a.top);
        }
        __syncthreads();
    }
    sum.join_wave();
    for (int o = 32; o; o /= 2) above += __shfl_xor(above, o, 64);
    meet();
    if (w == 0) logprobs_finish(a, row, sum, xt, above, best.key);
}

#define RT_LOGPROBS_KERNELS(S, T)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) k_logprobs_##S(LogprobsArgs a) { logprobs<T, false>(a); } \
    extern "C" __global__ void __launch_bounds__(256) k_logprobs_top_##S(LogprobsArgs a) { logprobs<T, true>(a); }
RT_LOGPROBS_KERNELS(f32, float)
RT_LOGPROBS_KERNELS(f16, _Float16)
