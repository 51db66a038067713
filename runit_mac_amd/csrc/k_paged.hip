// k_paged.hip — a batch of sequences over paged key / value caches of f32 or
// f16: the rotary embedding with the append of new rows, their way back, and the
// causal attention (rt_paged.h and, of f16 pages, its wide blocks); pages of
// any type copied.
#include "rt_paged.h"

// ───────────────────────────── append ─────────────────────────────
//
// One workgroup a row and group of heads: its first HD/2 threads make the
// row's cosines and sines while the heads' loads are on their way.  The angle's
// turns are reduced in 64 bits: position · θ^(-2d/HD) in 32 would be off by
// 2^-24 of itself, half a percent of a radian at position 100,000.  Bound by
// the rows' bytes: 2,068 rows of 28 + 2·4 heads of 128 into f16 pages
// (72 MB) 15 µs = 4.8 TB/s; few rows, by the launch (2.3 µs).
template <int HD, class T>
RT_DEV void store4(T* p, f32x4 v) {
    if constexpr (sizeof(T) == 4) {
        *(f32x4*)p = v;
    } else {
        h4_t h;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) h[i] = (_Float16)v[i];  // (nearest even)
        *(h4_t*)p = h;
    }
}
template <int HD, class T>
RT_DEV void paged_append(const PagedAppendArgs& a) {
    constexpr uint32_t half = HD / 2, TH = half / 4, HW = 256 / TH;  // threads a head, heads a pass
    __shared__ float cs[half], sn[half];
    const PagedBatch& b = a.b;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, ht = tid / TH, d = tid % TH * 4;
    const uint32_t s = paged_seq(b, row);
    if (s >= b.n_seqs) return;  // behind the last sequence
    const auto [pos, page] = paged_place(b, s, row);
    paged_turns<HD>(pos, a.log2_theta, cs, sn);
    __syncthreads();
    const uint32_t slot = pos & ((1u << b.ps_shift) - 1);
    f32x4 c4, s4;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) c4[i] = cs[d + i], s4[i] = sn[d + i];
    const uint32_t heads = a.H + 2 * b.KVH;
    for (uint32_t h = blockIdx.y * HW + ht; h < heads; h += gridDim.y * HW) {
        const bool isq = h < a.H, isv = h >= a.H + b.KVH;
        const uint32_t kh = isq ? h : isv ? h - a.H - b.KVH : h - a.H;
        const float* src = (isq ? a.q + ((size_t)row * a.H + kh) * HD : (isv ? a.v : a.k) + ((size_t)row * b.KVH + kh) * HD) + d;
        const f32x4 lo = *(const f32x4*)src, hi = *(const f32x4*)(src + half);
        f32x4 x = lo, y = hi;
        if (!isv) {
            x = lo * c4 - hi * s4;
            y = lo * s4 + hi * c4;
        }
        if (isq) {
            float* o = a.q_out + ((size_t)row * a.H + kh) * HD + d;
            *(f32x4*)o = x;
            *(f32x4*)(o + half) = y;
        } else if (page < b.num_pages) {
            T* o = (T*)(isv ? b.v : b.k) + page * b.page_stride + (((size_t)kh << b.ps_shift) + slot) * HD + d;
            store4<HD, T>(o, x);
            store4<HD, T>(o + half, y);
        }
    }
}

// o = Σ o_c·2^(m_c − M) / Σ l_c·2^(m_c − M) over a row's chunks, in their order,
// the prefix's after the sequence's own
template <int HD, bool WIDE>
RT_DEV void paged_merge(const PagedAttnArgs& a) {
    constexpr uint32_t TH = HD / 4, SR = paged_slot_rows<WIDE>();
    const PagedBatch& b = a.b;
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, rh = i / TH, d = i % TH * 4;
    const uint32_t rows = b.row_start ? min(b.row_start[b.n_seqs], b.rows) : min(b.n_seqs, b.rows);
    if (rh >= rows * a.H) return;
    const uint32_t kvh = rh % a.H / (a.H / b.KVH);
    typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
    const u4_t in = *(const u4_t*)(a.info + (size_t)rh * 4);
    const uint32_t n0 = in[1] / SR, n = n0 + (a.shared_len ? in[3] / SR : 0);
    if (!a.shared_len && n0 == 1) return;  // (written whole)
    if (in[0] >= a.jobs || n0 > a.jobs - in[0] || n > n0 && (in[2] >= a.jobs || n - n0 > a.jobs - in[2])) return;
    const float NEG = -__builtin_huge_valf();
    float M = NEG, L = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    // BATCH chunks from x0 on, all on their way together
    auto take = [&]<uint32_t BATCH>(uint32_t x0) {
        float mc[BATCH], lc[BATCH], mx = M;
        f32x4 oc[BATCH];
#pragma unroll
        for (uint32_t u = 0; u < BATCH; ++u) {
            const uint32_t x = min(x0 + u, n - 1), job = x < n0 ? in[0] + x : in[2] + x - n0;
            const size_t slot = ((size_t)job * b.KVH + kvh) * SR + (x < n0 ? in[1] : in[3]) % SR;
            mc[u] = a.ml[2 * slot], lc[u] = a.ml[2 * slot + 1];
            oc[u] = *(const f32x4*)(a.part + slot * HD + d);
        }
#pragma unroll
        for (uint32_t u = 0; u < BATCH; ++u) mx = fmaxf(mx, mc[u]);
        const float md = mx == NEG ? 0.0f : mx, f0 = __builtin_amdgcn_exp2f(M - md);
        M = mx;
        L *= f0;
        o *= f0;
#pragma unroll
        for (uint32_t u = 0; u < BATCH; ++u) {
            if (x0 + u >= n) continue;
            const float f = __builtin_amdgcn_exp2f(mc[u] - md);
            L = fmaf(f, lc[u], L);
            o += f * oc[u];
        }
    };
    // (a prefix has tens of chunks: 40 rows over 8,192 positions 6.5 µs eight at a time, 8.0 four; a sequence's few
    // 9.4 and 7.8)
    if (a.shared_len)
        for (uint32_t x0 = 0; x0 < n; x0 += 8) take.template operator()<8>(x0);
    else
        for (uint32_t x0 = 0; x0 < n; x0 += 4) take.template operator()<4>(x0);
    *(f32x4*)(a.out + (size_t)rh * HD + d) = L == 0.0f ? f32x4{0, 0, 0, 0} : o / L;
}

#define RT_PAGED_KERNELS(HD)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) k_paged_append_f32_hd##HD(PagedAppendArgs a) {     \
        paged_append<HD, float>(a);                                                                       \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) k_paged_append_f16_hd##HD(PagedAppendArgs a) {     \
        paged_append<HD, _Float16>(a);                                                                    \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) k_paged_attn_f32_hd##HD(PagedAttnArgs a) {      \
        paged_attn<HD, float, false>(a);                                                                  \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) k_paged_attn_f16_hd##HD(PagedAttnArgs a) {      \
        paged_attn<HD, _Float16, false>(a);                                                               \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) k_paged_attn_f16w_hd##HD(PagedAttnArgs a) {     \
        paged_attn<HD, _Float16, true>(a);                                                                \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) k_paged_merge_hd##HD(PagedAttnArgs a) {            \
        paged_merge<HD, false>(a);                                                                        \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) k_paged_mergew_hd##HD(PagedAttnArgs a) {           \
        paged_merge<HD, true>(a);                                                                         \
    }
RT_PAGED_KERNELS(64)
RT_PAGED_KERNELS(128)
RT_PAGED_KERNELS(256)

// ───────────────────────────── rows read back ─────────────────────────────

template <class T, class O>
RT_DEV void paged_gather_plain(const PagedGatherArgs& a) {
    typedef T t4_t __attribute__((ext_vector_type(4)));
    paged_gather<O>(a, [&](uint32_t page, uint32_t kvh, uint32_t slot, bool isv, uint32_t d) {
        const T* p = (const T*)(isv ? a.b.v : a.b.k) + page * a.b.page_stride + (((size_t)kvh << a.b.ps_shift) + slot) * a.head_dim;
        return __builtin_convertvector(*(const t4_t*)(p + d), f32x4);
    });
}
#define RT_PAGED_GATHER(S, T, OS, O) \
    extern "C" __global__ void __launch_bounds__(256) k_paged_gather_##S##_##OS(PagedGatherArgs a) { paged_gather_plain<T, O>(a); }
RT_PAGED_GATHER(f32, float, f32, float)
RT_PAGED_GATHER(f32, float, f16, _Float16)
RT_PAGED_GATHER(f16, _Float16, f32, float)
RT_PAGED_GATHER(f16, _Float16, f16, _Float16)

// ───────────────────────────── pages copied ─────────────────────────────
//
// Entry i makes page dst[i] of every pool a copy of page src[i], as if one after
// another.  A workgroup has a slice of one page of one pool, or (SMALL) a page of several
// pools (2,000 pages of 1,152 bytes in 48 pools 45 µs, of one pool each 120), its entry alone where
// that shares no page with another entry but a source with sources (the scan
// of the lists goes on while the slice is on its way).  Entries that do, a chain or
// a page written twice, are the first of them's: it copies its slice of all of
// them in order, every byte by one thread, which sees its own stores.
// Bound by the pages' bytes: 277 pages of 18 KB in 56 pools 109 µs, 5.2 TB/s read and
// written (a large copy makes 5.1); 8 pages of 16 KB in 48 pools 5.0 µs, a launch.
template <bool SMALL>
RT_DEV void paged_copy(const PagedCopyArgs& a) {
    const uint32_t tid = threadIdx.x, i = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const uint32_t b0 = slice * a.slice_bytes, bytes = min(a.page_bytes - b0, a.slice_bytes);
    uint8_t* pool = (uint8_t*)a.pools[SMALL ? 0 : blockIdx.y] + b0;
    auto entry = [&](uint32_t j, uint32_t& s, uint32_t& d) {
        s = a.src[j], d = a.dst[j];
        return s < a.num_pages && d < a.num_pages;
    };
    uint32_t s, d;
    if (!entry(i, s, d)) return;
    // whether entry j (pages s, d) meets another; the whole workgroup's answer
    auto meets = [&](uint32_t j, uint32_t s, uint32_t d) {
        bool hit = false;
#pragma unroll 4
        for (uint32_t k = tid; k < a.n; k += 256) {
            uint32_t s2, d2;
            hit |= entry(k, s2, d2) && k != j && (d2 == d || d2 == s || s2 == d);
        }
        return __syncthreads_or(hit);
    };
    // (the slice is on its way while the lists are looked through)
    constexpr uint32_t V = RT_COPY_SLICE / (256 * 16);
    u32x4 v[V];
    uint8_t* at[V];  // (small pages) in page 0; null: nothing
    if constexpr (SMALL) {
        const uint32_t p0 = blockIdx.y * a.group, pools = min(a.n_pools - p0, a.group);
#pragma unroll
        for (uint32_t u = 0; u < V; ++u) {
            const uint32_t o = (256 * u + tid) * 16, p = o / bytes;
            at[u] = p < pools ? (uint8_t*)a.pools[p0 + p] + (o - p * bytes) : nullptr;
        }
    }
    auto load = [&](uint32_t s) {
        const uint8_t* from = pool + s * a.page_stride;
#pragma unroll
        for (uint32_t u = 0; u < V; ++u) {
            const uint32_t o = (256 * u + tid) * 16;
            if (SMALL ? at[u] != nullptr : o < bytes) v[u] = *(const u32x4*)(SMALL ? at[u] + s * a.page_stride : from + o);
        }
    };
    auto store = [&](uint32_t d) {
        uint8_t* to = pool + d * a.page_stride;
#pragma unroll
        for (uint32_t u = 0; u < V; ++u) {
            const uint32_t o = (256 * u + tid) * 16;
            if (SMALL ? at[u] != nullptr : o < bytes) *(u32x4*)(SMALL ? at[u] + d * a.page_stride : to + o) = v[u];
        }
    };
    load(s);
    if (!meets(i, s, d)) {
        if (s != d) store(d);
        return;
    }
    for (uint32_t j = 0; j < i; ++j) {
        uint32_t s2, d2;
        if (entry(j, s2, d2) && meets(j, s2, d2)) return;  // (an earlier one does it)
    }
    for (uint32_t j = i; j < a.n; ++j) {
        uint32_t s2, d2;
        if (entry(j, s2, d2) && s2 != d2 && meets(j, s2, d2)) load(s2), store(d2);
    }
}
extern "C" __global__ void __launch_bounds__(256) k_paged_copy(PagedCopyArgs a) { paged_copy<false>(a); }
extern "C" __global__ void __launch_bounds__(256) k_paged_copy_small(PagedCopyArgs a) { paged_copy<true>(a); }
