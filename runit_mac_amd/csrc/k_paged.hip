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

template <int HD>
RT_DEV void paged_wide(const PagedAttnArgs& a, const PagedCols<HD, _Float16>& co, const PagedJob& j, uint32_t job,
                       h8_t* lds) {
    typedef PagedStage<HD> Stage;
    typedef PagedAcc<HD, _Float16> Acc;
    typedef short s4_t __attribute__((ext_vector_type(4)));
    typedef float f16v __attribute__((ext_vector_type(16)));
    typedef __attribute__((address_space(3))) s4_t* tptr_t;
    constexpr uint32_t NW = RT_PAGED_WAVES, SR = RT_PAGED_WIDE_ROWS, KS = HD / 16, NB = HD / 32;
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t c = lane & 31, h = lane >> 5;  // column; of its positions and elements 4h .. of every 8
    const float NEG = -__builtin_huge_valf(), scale2 = a.scale * 1.44269504f;
    PagedView<_Float16> v = co.v;
    const bool idle = 32 * w >= co.ncl;  // (brings tiles, computes none)
    const uint32_t limx = co.pre ? co.hi : __builtin_amdgcn_readfirstlane(co.lim(co.ncl - 1));
    v.t1 = min(v.t1, limx > v.lo ? (limx + RT_PAGED_TILE - 1) / RT_PAGED_TILE - v.tb : 0u);
    const uint32_t t0 = 2 * j.chunk, step = 2 * j.chunks;
    const uint32_t turns = t0 < v.t1 ? (v.t1 - t0 + step - 1) / step : 0;
    // where the two tiles of 64 turns are, one turn a lane, from the KV head's part of the pool on (~0:
    // nowhere).  Scalar loads in the loop would hold up its LDS reads, which share their counter.
    uint64_t at[2];
    auto ids_from = [&](uint32_t i0) {
        const uint32_t t = t0 + (i0 + lane) * step;
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
            const uint32_t page =
                i0 + lane < turns && t + u < v.t1 ? v.table[(v.tb + t + u) * RT_PAGED_TILE >> v.ps_shift] : v.num_pages;
            at[u] = page < v.num_pages ? v.place(t + u, page, HD) * 2 : ~0ull;
        }
    };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const h8_t*)lds);
    // a wave's parts of a stage, 64 pieces each: what its lanes read from a tile's place on
    const uint8_t* src[Stage::LOADS];
#pragma unroll
    for (uint32_t x = 0; x < Stage::LOADS; ++x) {
        const uint32_t n = (x * NW + w) * 64 + lane, r = n / Stage::ROW, p = n % Stage::ROW;
        // (the permutation undoes itself)
        src[x] = (const uint8_t*)((r < 32 ? v.k : v.v) + (size_t)(r & 15) * HD + (Stage::piece(r, p) - r * Stage::ROW) * 8);
    }
    // turn i's tiles into stage i % N; whether they have a page, a bit each
    auto bring = [&](uint32_t i) {
        uint64_t off[2];
        uint32_t there = 0;
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
            const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)at[u], i & 63);
            const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(at[u] >> 32), i & 63);
            there |= hi != 0xffffffffu ? 1u << u : 0u;
            off[u] = hi != 0xffffffffu ? (uint64_t)hi << 32 | lo : 0;  // (nowhere: the pool's first page)
        }
        const uint32_t st = lds0 + i % Stage::N * Stage::LEN * 16;
#pragma unroll
        for (uint32_t x = 0; x < Stage::LOADS; ++x) {
            const uint32_t n = (x * NW + w) * 64;
            bring16(src[x] + (n / Stage::ROW & 16 ? off[1] : off[0]), st + n * 16);
        }
        return there;
    };
    // the block's queries into all stages, a wave's 32 KB·HD / 256 in its own quarter, each instruction whole rows of
    // them: lanes that read and wrote their columns' pieces themselves took 3 µs more of the prompt chunks' 57
    constexpr uint32_t PC = HD / 4, QL = HD / 8;  // 16-byte pieces a column, instructions a wave
    h8_t* own = lds + w * 32 * PC;
    const uint32_t cc = min(32 * w + c, co.ncl - 1), rh = co.row(cc) * a.H + co.head(cc);
    auto piece = [&](uint32_t col, uint32_t p) { return col * PC + (p ^ (col & 15)); };  // (16 columns' same one: all banks)
    ids_from(0);
#pragma unroll 2
    for (uint32_t x = 0; x < QL; ++x) {
        const uint32_t col = (64 * x + lane) / PC, p = lane % PC;
        bring16(a.q + (size_t)__shfl(rh, col, 64) * HD + 4 * (piece(col, p) - col * PC),
                lds0 + (w * 32 * PC + 64 * x) * 16);
    }
    // the column's limit, and what the last (the most) and the first of the wave's see
    const uint32_t lim = co.lim(cc);
    uint32_t limx_w = lim, limn_w = lim;
    for (uint32_t o = 1; o < 32; o *= 2) {
        limx_w = max(limx_w, __shfl_xor(limx_w, o, 64));
        limn_w = min(limn_w, __shfl_xor(limn_w, o, 64));
    }
    limx_w = __builtin_amdgcn_readfirstlane(limx_w);
    limn_w = __builtin_amdgcn_readfirstlane(limn_w);
    // the query: elements 16n + 8h .. of column c
    h8_t qh[KS], ql[KS];
    float qs;
    {
        stages_left<Stage::LOADS>(0);
        asm volatile("" ::: "memory");
        float x[KS][8], mx = 0.0f;
#pragma unroll
        for (uint32_t n = 0; n < KS; ++n)
#pragma unroll
            for (uint32_t e = 0; e < 8; e += 4) {
                const f32x4 y = *(const f32x4*)(own + piece(c, 4 * n + 2 * h + e / 4)) * scale2;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    x[n][e + k] = y[k];
                    mx = fmaxf(mx, fabsf(y[k]));
                }
            }
        qs = split_query<KS>(x, fmaxf(mx, __builtin_bit_cast(float, lane_xor<32>(__builtin_bit_cast(uint32_t, mx)))), qh, ql);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4 | 0 << 8);  // (the queries are read before tiles come)
    __builtin_amdgcn_s_barrier();
    uint32_t here = 0;  // bring()'s bits of turns i .. i + 3
#pragma unroll
    for (uint32_t i = 0; i < Stage::N - 1; ++i)
        if (i < turns) here |= bring(i) << 2 * i;
    // where in a stage the lane's values of elements 32n .. are (of positions 16x + 8k .., as many rows on: the
    // permutation goes by the row's last bits)
    uint32_t vat[NB];
#pragma unroll
    for (uint32_t n = 0; n < NB; ++n)
        vat[n] = Stage::piece(32 + 4 * h + (lane >> 2 & 3), 4 * n + (lane >> 3 & 2) + (lane >> 1 & 1)) * 16 + (lane & 1) * 8;
    f16v o[NB];
#pragma unroll
    for (uint32_t n = 0; n < NB; ++n) o[n] = f16v{};
    float m = NEG, l = 0.0f;
    for (uint32_t i = 0; i < turns; ++i) {
        const uint32_t p0 = (v.tb + t0 + i * step) * RT_PAGED_TILE;
        const uint32_t there = here & 3;
        h8_t* st = lds + i % Stage::N * Stage::LEN;
        stages_left<Stage::LOADS>(turns - 1 - i);
        __builtin_amdgcn_s_barrier();  // (this stage is there, the one before is read)
        asm volatile("" ::: "memory");
        here >>= 2;
        if (i + Stage::N - 1 < turns) {
            const uint32_t in = i + Stage::N - 1;
            if (in % 64 == 0) ids_from(in);
            here |= bring(in) << 4;
        }
        if (p0 < v.lo || p0 + 2 * RT_PAGED_TILE > limx || there != 3) {
            // positions that no column sees may hold anything: zeros
            for (uint32_t n = tid; n < 32 * Stage::ROW; n += 64 * NW) {
                const uint32_t r = n / Stage::ROW;
                if (p0 + r < v.lo || p0 + r >= limx || !(there >> r / 16 & 1)) st[32 * Stage::ROW + n] = h8_t{};
            }
            __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4 | 0 << 8);  // (LDS)
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        }
        if (!idle && p0 < limx_w) {
            f16v s = {};
#pragma unroll
            for (uint32_t n = 0; n < KS; ++n) {
                const h8_t k = st[Stage::piece(c, 2 * n + h)];
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[n], s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[n], s, 0, 0, 0);
            }
            float p[16];  // of the positions 8(r / 4) + 4h + r % 4
#pragma unroll
            for (uint32_t r = 0; r < 16; ++r) p[r] = s[r];
            if (p0 < v.lo || p0 + 2 * RT_PAGED_TILE > limn_w || there != 3) {
#pragma unroll
                for (uint32_t r = 0; r < 16; ++r) {
                    const uint32_t pos = p0 + 8 * (r / 4) + 4 * h + r % 4;
                    if (pos < v.lo || pos >= lim || !(there >> r / 8 & 1)) p[r] = NEG;
                }
            }
            float tmax = p[0];
#pragma unroll
            for (uint32_t r = 1; r < 16; ++r) tmax = fmaxf(tmax, p[r]);
            tmax = fmaxf(tmax, __builtin_bit_cast(float, lane_xor<32>(__builtin_bit_cast(uint32_t, tmax)))) * qs;
            if (__ballot(tmax > m + Acc::GROW)) {
                const float mn = fmaxf(m, tmax), f = __builtin_amdgcn_exp2f(m - (mn == NEG ? 0.0f : mn));
                m = mn;
                l *= f;
#pragma unroll
                for (uint32_t n = 0; n < NB; ++n) o[n] *= f;
            }
            const float md = (m == NEG ? 0.0f : m) - Acc::BIAS;
#pragma unroll
            for (uint32_t r = 0; r < 16; ++r) {
                p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], qs, -md));
                l += p[r];
            }
            h8_t ph[2], pl[2];
            split_weights(p, ph[0], pl[0]);
            split_weights(p + 8, ph[1], pl[1]);
            const uint32_t vst = lds0 + i % Stage::N * Stage::LEN * 16;
#pragma unroll
            for (uint32_t n = 0; n < NB; ++n)
#pragma unroll
                for (uint32_t x = 0; x < 2; ++x) {
                    s4_t y[2];  // element 32n + c of the positions 16x + 4h .., and eight on
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k)
                        y[k] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (tptr_t)(uintptr_t)(vst + vat[n] + (16 * x + 8 * k) * Stage::ROW * 16));
                    const h8_t vv = __builtin_bit_cast(h8_t, __builtin_shufflevector(y[0], y[1], 0, 1, 2, 3, 4, 5, 6, 7));
                    o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv, ph[x], o[n], 0, 0, 0);
                    o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vv, pl[x], o[n], 0, 0, 0);
                }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4 | 0 << 8);  // (its reads are done before the next barrier)
    }
    __builtin_amdgcn_s_barrier();  // (all stages are read)
    if (idle) return;
    const bool alone = j.chunks == 1 && !a.shared_len;
    l += __builtin_bit_cast(float, lane_xor<32>(__builtin_bit_cast(uint32_t, l)));
    bool bad = !(l < __builtin_huge_valf());
#pragma unroll
    for (uint32_t n = 0; n < NB; ++n)
#pragma unroll
        for (uint32_t r = 0; r < 16; ++r) bad |= !(fabsf(o[n][r]) < __builtin_huge_valf());
    if (!__ballot(bad)) {
        // through the wave's quarter, so that a row leaves whole
        const float f = !alone ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (uint32_t n = 0; n < NB; ++n)
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x)
                *(f32x4*)(own + piece(c, 8 * n + 2 * x + h)) =
                    f32x4{o[n][4 * x], o[n][4 * x + 1], o[n][4 * x + 2], o[n][4 * x + 3]} * f;
        asm volatile("" ::: "memory");
        float* part = co.template place<SR>(job, 32 * w, false);
#pragma unroll 2
        for (uint32_t x = 0; x < QL; ++x) {
            const uint32_t col = (64 * x + lane) / PC, p = lane % PC;
            const f32x4 y = *(const f32x4*)(own + piece(col, p));
            float* to = alone ? a.out + (size_t)__shfl(rh, col, 64) * HD : part + col * HD;
            if (32 * w + col < co.ncl) *(f32x4*)(to + 4 * p) = y;
        }
        if (32 * w + c < co.ncl && h == 0) co.template state<SR>(j, job, cc, m, l, alone);
        return;
    }
#pragma unroll 1
    for (uint32_t u = 0; u < 2; ++u) {  // 16 columns at a time
        const uint32_t c1 = 32 * w + 16 * u + (lane & 15), c2 = min(c1, co.ncl - 1);
        if (32 * w + 16 * u >= co.ncl) break;
        Acc acc;
        paged_f32<HD, _Float16, 2>(acc, v, co.q(c2), scale2, t0, step, co.lim(c2), limn_w, limx_w);
        co.template put<SR>(acc, j, job, c1, alone);
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
// another.  A workgroup has a slice of one page of one pool, its entry alone where
// that shares no page with another entry but a source with sources (the scan
// of the lists goes on while the slice is on its way).  Entries that do, a chain or
// a page written twice, are the first of them's: it copies its slice of all of
// them in order, every byte by one thread, which sees its own stores.
// Bound by the pages' bytes.
RT_DEV void paged_copy(const PagedCopyArgs& a) {
    const uint32_t tid = threadIdx.x, i = blockIdx.x / a.slices, slice = blockIdx.x % a.slices;
    const uint32_t b0 = slice * a.slice_bytes, b1 = min(a.page_bytes, b0 + a.slice_bytes);
    uint8_t* pool = (uint8_t*)a.pools[blockIdx.y];
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
    auto load = [&](uint32_t s) {
        const uint8_t* from = pool + s * a.page_stride;
#pragma unroll
        for (uint32_t u = 0; u < V; ++u) {
            const uint32_t o = b0 + (256 * u + tid) * 16;
            if (o < b1) v[u] = *(const u32x4*)(from + o);
        }
    };
    auto store = [&](uint32_t d) {
        uint8_t* to = pool + d * a.page_stride;
#pragma unroll
        for (uint32_t u = 0; u < V; ++u) {
            const uint32_t o = b0 + (256 * u + tid) * 16;
            if (o < b1) *(u32x4*)(to + o) = v[u];
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
extern "C" __global__ void __launch_bounds__(256) k_paged_copy(PagedCopyArgs a) { paged_copy(a); }
