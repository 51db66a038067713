// k_paged.hip — a batch of sequences over paged key / value caches: the rotary
// embedding with the append of new rows, and the causal attention.
//
// A page holds [KV heads][page size][head size] keys (values), f32 or f16, and
// a sequence's position j is in page table[s][j / page size].  A page id that
// is none of the pool's is no page: its positions are neither stored nor seen.
// Sequence s has the rows row_start[s] .. row_start[s + 1], at its last
// positions: row i of n at kv_len − n + i.  Lengths, rows and tables are read on
// the device, so that a captured graph follows them.
#include "rt_attn.h"

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h4_t __attribute__((ext_vector_type(4)));

// rows of sequence s: the first and their number (0 where the list is not in order)
struct SeqRows {
    uint32_t first, n;
};
RT_DEV SeqRows seq_rows(const PagedBatch& b, uint32_t s) {
    if (!b.row_start) return {s, s < b.rows ? 1u : 0u};
    const uint32_t r0 = min(b.row_start[s], b.rows), r1 = min(b.row_start[s + 1], b.rows);
    return {r0, r1 > r0 ? r1 - r0 : 0u};
}

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
    __shared__ uint32_t seq_s;
    const PagedBatch& b = a.b;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, ht = tid / TH, d = tid % TH * 4;
    // the row's sequence
    uint32_t s = row;
    if (b.row_start) {
        if (tid == 0) seq_s = b.n_seqs;
        __syncthreads();
        for (uint32_t i = tid; i < b.n_seqs; i += 256)
            if (b.row_start[i] <= row && row < b.row_start[i + 1]) seq_s = i;
        __syncthreads();
        s = seq_s;
    }
    if (s >= b.n_seqs) return;  // behind the last sequence
    const SeqRows sr = seq_rows(b, s);
    const uint32_t back = sr.n - (row - sr.first), len = b.kv_len[s];  // the row is the back-th from the end
    const bool there = back <= len;
    const uint32_t pos = there ? len - back : 0;
    if (tid < half) {
        const double turns = (double)pos * exp2(-(double)(2 * tid) / HD * a.log2_theta) * 0.15915494309189535;
        const float t = (float)(2.0 * (turns - rint(turns)));
        sincospif(t, &sn[tid], &cs[tid]);
    }
    __syncthreads();
    const uint32_t pi = pos >> b.ps_shift, slot = pos & ((1u << b.ps_shift) - 1);
    const uint32_t page = there && pi < b.table_stride ? b.table[(size_t)s * b.table_stride + pi] : b.num_pages;
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

// ───────────────────────────── attention ─────────────────────────────
//
// The rows of a sequence's KV head — (row, head of the group) pairs, row-major
// — are columns of Sᵀ = K·Qᵀ and Oᵀ = Vᵀ·Pᵀ on the matrix cores: a lane has four
// positions of one column in registers, in the order that the second product
// takes them, so that scores never leave their registers.  A job is a block of
// columns over a chunk of tiles of 16 positions, one workgroup.  Chunks take
// tiles in turn, so that those of a sequence read one window of it together.
//
// Narrow blocks (16 columns; decoding rows): the four waves take the chunk's
// tiles in turn, keys and values straight from the pages into registers, each
// with a softmax of its own, and meet in LDS.  Bound by the pages' bytes: 24
// sequences of up to 8,000 positions, 4 KV heads of 128, f16 (182 MB) 41.7 µs
// = 4.4 TB/s; one of 100,003, f32 (410 MB) 79 µs = 5.2 TB/s; a large copy
// makes 5.1.  A few hundred positions: 8.3 µs, of which the launch and the
// planning are 4, two trips to memory and the meeting the rest.
// Wide blocks (f16 pages; prompt chunks, a shared prefix): each of four waves has
// 32 columns of its own and all take every tile, from LDS, on the 32x32x16 f16
// matrix cores.  Bound by these and the vector operations beside them, 32 and
// some 140 a turn of 32 positions: 1.88 µs a turn of all workgroups, two a CU,
// = 1.14 PFLOP/s of products (a large f16 product makes 1.10).  Of its 4,500
// cycles 32 products with 100 and 200 such operations alone take 2,800 and 3,300,
// the products 2,500 (measured).  What the rest goes to was not found: half as
// many barriers, fewer vector operations, other orders and priorities change
// nothing.  Planning, queries and parts: 10 µs a launch.
// Prompt chunks of 644 rows of 28 heads over 245 .. 4,005 positions 55 µs, 40
// rows over a shared prefix of 8,192 35 µs, with the parts' launch of 8 and 6 µs;
// the 16x16x32 form, with twice the products to issue and two columns' statistics
// a lane, took 3 % longer, blocks of 16 columns alone 280 and 118.
//
// f32 pages use the f32 matrix cores.  f16 pages use the f16 ones, keys and
// values as they are, queries and weights as pairs of f16 (x = hi + lo: 22
// bits): queries scaled by a power of two to [2^14, 2^15) a column, weights so
// that the largest is between 2^12 and 2^15: those down to 2^-14 of it keep
// their 22 bits, smaller ones are off by at most 2^-37 of it.  A job whose sums
// come out not finite (a value that is not, in places that only some of its
// columns see; the pairs make NaN of ∞ too) is computed again on the f32 matrix
// cores.
//
// The scale (1 / (√HD·ln 2)) comes before the maximum, one rounding: f32 scores
// take it as they leave the first product, f16 queries before they are split, and
// scores are in units of log 2 times a power of two.  So the reference is one of
// them, and a weight's exponent the difference of two rounded scores.  Scaled in
// the exponent's fma, the reference would be rounded apart from the scores: a factor of
// 2^16 at scores of 2^28, more than f32 holds from 2^32 on.  (f32 queries scaled
// instead hold up the first tile: 8.7 µs for 8.4 at a few hundred positions.)

template <bool WIDE>
constexpr uint32_t paged_slot_rows() { return WIDE ? RT_PAGED_WIDE_ROWS : RT_PAGED_ROWS; }

// The jobs of one KV head: blocks × chunks of every sequence in turn (and, with
// a shared prefix, before them those of all rows over it).  The chunk length
// comes from the work that the device finds, so that the jobs are alike
// whatever the lengths: jobs ≤ blocks + target.
struct PagedJob {
    uint32_t seq;             // n_seqs: the shared prefix
    uint32_t rb, chunk, first, chunks;  // block, chunk, first job of the block, its chunks
    uint32_t row0, rows, kv;  // the sequence's rows and length (prefix: all rows, its length)
    uint32_t len;             // tiles of a chunk (at most)
    bool any;
};
RT_DEV uint32_t paged_tiles(const PagedAttnArgs& a, uint32_t kv) {  // own tiles of a sequence of kv positions
    const uint32_t cap = a.b.table_stride << a.b.ps_shift, L = min(kv, cap);
    const uint32_t t0 = a.shared_len / RT_PAGED_TILE;
    const uint32_t t1 = (L + RT_PAGED_TILE - 1) / RT_PAGED_TILE;
    return L > a.shared_len ? t1 - t0 : 0;
}
// columns of a block of a sequence (or of all rows) with so many
template <bool WIDE>
RT_DEV uint32_t paged_block(uint32_t cols) { return WIDE && cols > 32 ? paged_slot_rows<WIDE>() : RT_PAGED_ROWS; }
RT_DEV uint32_t wave_scan_add(uint32_t v) {  // inclusive
    constexpr int ROW_SHR = 0x110, ROW_BCAST15 = 0x142, ROW_BCAST31 = 0x143;
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ROW_SHR + 1, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ROW_SHR + 2, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ROW_SHR + 4, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ROW_SHR + 8, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ROW_BCAST15, 0xA, 0xF, false);  // rows 1, 3: the one below's
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ROW_BCAST31, 0xC, 0xF, false);  // rows 2, 3: the lower half's
    return v;
}
// ceil(t / d), at least 1, for t < 2^24 and inv = 1 / d
RT_DEV uint32_t ceil_div(uint32_t t, uint32_t d, float inv) {
    uint32_t q = (uint32_t)((float)t * inv);  // off by one at most
    q -= q && q * d >= t ? 1u : 0u;
    q += q * d < t ? 1u : 0u;
    q += q * d < t ? 1u : 0u;
    return max(1u, q);
}
template <int HD, class T, bool WIDE>
RT_DEV PagedJob paged_job(const PagedAttnArgs& a, uint32_t job) {
    constexpr uint32_t STEP = sizeof(T) == 2 ? 2 : 1;  // (f16 pages: tiles in pairs)
    const uint32_t lane = threadIdx.x & 63, G = a.H / a.b.KVH, n = a.b.n_seqs;
    auto blocks_of = [&](uint32_t rows) {
        const uint32_t bc = paged_block<WIDE>(rows * G);
        return (rows * G + bc - 1) / bc;
    };
    // a lane's sequence: its rows, length, blocks and tiles
    uint32_t mb = 0, mt = 0, mkv = 0;
    SeqRows mr = {0, 0};
    auto look = [&](uint32_t s) {
        mr = s < n ? seq_rows(a.b, s) : SeqRows{0, 0};
        mkv = s < n ? a.b.kv_len[s] : 0;
        mb = blocks_of(mr.n);
        mt = paged_tiles(a, mkv);
    };
    look(lane);
    uint32_t pb = 0, pt = 0, all = 0;
    if (a.shared_len) {
        all = a.b.row_start ? min(a.b.row_start[n], a.b.rows) : min(n, a.b.rows);
        pb = blocks_of(all);
        pt = (a.shared_len + RT_PAGED_TILE - 1) / RT_PAGED_TILE;
    }
    float work = (float)mb * (float)mt;
    for (uint32_t s = lane + 64; s < n; s += 64) {
        look(s);
        work += (float)mb * (float)mt;
    }
    work = group_sum(work, 64) + (float)pb * (float)pt;
    work = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, work)));
    if (n > 64) look(lane);
    PagedJob j{};
    // (a thousandth more than the share: the sum's roundings leave no job over)
    const float share = a.target ? work * 1.001f / (float)a.target : 16777216.0f;
    j.len = share < 16777216.0f ? ((uint32_t)share + STEP) / STEP * STEP : 16777216u;
    if (j.len <= a.min_chunk) {
        j.len = a.min_chunk;
    } else if (n <= 64 && a.target) {
        // the shortest chunk, of 64 from an even share on, whose jobs are no more
        // than the resident workgroups
        const uint32_t c0 = max(a.min_chunk, ((uint32_t)(work / (float)a.slots) + STEP) / STEP * STEP);
        const uint32_t cl = c0 + lane * max(STEP, c0 / 128 / STEP * STEP);
        const float inv = 1.0f / (float)cl;
        auto about = [&](uint32_t t) { return fmaxf(1.0f, floorf(fmaf((float)t, inv, 0.9999f))); };
        float jobs = (float)pb * about(pt);
        // (a quarter of the sequences each wave)
        __shared__ float sums[RT_PAGED_WAVES][64];
        const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (w) jobs = 0.0f;
        for (uint32_t s = w; s < n; s += RT_PAGED_WAVES)
            jobs += (float)__builtin_amdgcn_readlane(mb, s) * about((uint32_t)__builtin_amdgcn_readlane(mt, s));
        sums[w][lane] = jobs;
        __syncthreads();
        jobs = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < RT_PAGED_WAVES; ++k) jobs += sums[k][lane];
        const uint64_t fit = __ballot(jobs <= (float)a.slots && cl < j.len);
        if (fit) {  // (counted exactly before it is taken)
            const uint32_t c1 = __builtin_amdgcn_readlane(cl, __builtin_ctzll(fit));
            const float inv1 = 1.0f / (float)c1;
            const uint32_t own = __builtin_amdgcn_readlane(wave_scan_add(mb * ceil_div(mt, c1, inv1)), 63);
            if (own + pb * ceil_div(pt, c1, inv1) <= a.slots) j.len = c1;
        }
    }
    if (!WIDE && !a.shared_len && a.target && n <= 64) {
        // no more than sixteen chunks, which meet in one trip, where that takes chunks twice as long at most
        // (nine sequences of up to 4,000 positions with drafts 17.8 -> 15.8 µs, sixteen decoding 13.8 -> 12.5)
        uint32_t most = mt;
        most = max(most, lane_xor<1>(most)), most = max(most, lane_xor<2>(most)), most = max(most, lane_xor<4>(most));
        most = max(most, lane_xor<8>(most)), most = max(most, lane_xor<16>(most)), most = max(most, lane_xor<32>(most));
        const uint32_t len = ((uint32_t)__builtin_amdgcn_readfirstlane(most) / 16 + STEP) / STEP * STEP;
        if (j.len < len && len <= 2 * j.len) j.len = len;
    }
    const float inv = 1.0f / (float)j.len;
    auto found = [&](uint32_t seq, uint32_t base, uint32_t nc) {
        const uint32_t k = job - base;
        j.seq = seq;
        j.rb = k / nc;
        j.chunk = k % nc;
        j.first = job - j.chunk;
        j.chunks = nc;
        j.any = true;
    };
    uint32_t base = 0;
    if (pb) {
        const uint32_t nc = ceil_div(pt, j.len, inv);
        if (job < pb * nc) {
            found(n, 0, nc);
            j.rows = all, j.kv = a.shared_len;
            return j;
        }
        base = pb * nc;
    }
    for (uint32_t s0 = 0; s0 < n; s0 += 64) {
        if (s0) look(s0 + lane);
        const uint32_t nc = ceil_div(mt, j.len, inv), mine = mb * nc;
        const uint32_t upto = base + wave_scan_add(mine);
        const uint64_t hit = __ballot(job < upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            found(s0 + l, (uint32_t)__builtin_amdgcn_readlane(upto - mine, l), (uint32_t)__builtin_amdgcn_readlane(nc, l));
            j.row0 = __builtin_amdgcn_readlane(mr.first, l), j.rows = __builtin_amdgcn_readlane(mr.n, l);
            j.kv = __builtin_amdgcn_readlane(mkv, l);
            return j;
        }
        base = (uint32_t)__builtin_amdgcn_readlane(upto, 63);
    }
    return j;
}

RT_DEV uint64_t pair_of(float lo, float hi) {
    return (uint64_t)__builtin_bit_cast(uint32_t, hi) << 32 | __builtin_bit_cast(uint32_t, lo);
}
RT_DEV float pair_lo(uint64_t p) { return __builtin_bit_cast(float, (uint32_t)p); }
RT_DEV float pair_hi(uint64_t p) { return __builtin_bit_cast(float, (uint32_t)(p >> 32)); }
RT_DEV f32x4 mfma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
RT_DEV f32x4 mfma32(h8_t a, h8_t b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// Where a job's columns and positions are.
template <class T>
struct PagedView {
    const T *k, *v;         // the KV head's part of page 0
    const uint32_t* table;
    uint64_t page_stride;
    uint32_t num_pages, ps_shift;
    uint32_t tb, t1;        // tile 0 of the job's numbering, the end
    uint32_t lo;            // first position seen
    RT_DEV uint32_t page(uint32_t t) const {  // t: the same in every lane; no page behind the end
        typedef const __attribute__((address_space(4))) uint32_t* sptr_t;  // (a scalar load)
        return t < t1 ? ((sptr_t)table)[(tb + t) * RT_PAGED_TILE >> ps_shift] : num_pages;
    }
    RT_DEV size_t place(uint32_t t, uint32_t page, uint32_t hd) const {
        return page * page_stride + (size_t)((tb + t) * RT_PAGED_TILE & ((1u << ps_shift) - 1)) * hd;
    }
};

// Operands of a tile.  Keys: lane l holds position l % 16, KW of every 4·KW
// elements from KW·(l / 16) on; values: of the positions 4(l / 16) + r, VW of
// every 16·VW elements from VW·(l % 16) on.
template <int HD, class T>
struct PagedTile {
    static constexpr uint32_t KW = sizeof(T) == 4 ? 4 : 8, KN = HD / (4 * KW);
    static constexpr uint32_t VW = sizeof(T) == 4 || HD == 64 ? 4 : 8, VN = HD / (16 * VW);
    typedef T kvec __attribute__((ext_vector_type(KW)));
    typedef T vvec __attribute__((ext_vector_type(VW)));
    kvec k[KN];
    vvec v[4][VN];
    RT_DEV void load_k(const T* kb, uint32_t lane) {
        const T* kp = kb + (size_t)(lane & 15) * HD + (lane >> 4) * KW;
#pragma unroll
        for (uint32_t i = 0; i < KN; ++i) k[i] = *(const kvec*)(kp + i * 4 * KW);
    }
    RT_DEV void load_v(const T* vb, uint32_t lane) {
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const T* vp = vb + (size_t)(4 * (lane >> 4) + r) * HD + (lane & 15) * VW;
#pragma unroll
            for (uint32_t i = 0; i < VN; ++i) v[r][i] = *(const vvec*)(vp + i * 16 * VW);
        }
    }
    RT_DEV void no_k() {
#pragma unroll
        for (uint32_t i = 0; i < KN; ++i) k[i] = kvec{};
    }
    RT_DEV void no_v() {
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r)
#pragma unroll
            for (uint32_t i = 0; i < VN; ++i) v[r][i] = vvec{};
    }
    // positions that no column sees may hold anything: zeros
    RT_DEV void clear(uint32_t pos0, uint32_t lo, uint32_t limx) {
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r)
#pragma unroll
            for (uint32_t i = 0; i < VN; ++i) v[r][i] = pos0 + r < lo || pos0 + r >= limx ? vvec{} : v[r][i];
    }
};

// over the four lanes of a column
RT_DEV float column_max(float v) {
    v = fmaxf(v, __builtin_bit_cast(float, lane_xor<16>(__builtin_bit_cast(uint32_t, v))));
    return fmaxf(v, __builtin_bit_cast(float, lane_xor<32>(__builtin_bit_cast(uint32_t, v))));
}

// 16 columns' running reference, near the maximum (in units of log 2), sum and outputs.  Lane (c =
// l % 16, g = l / 16) has column c's outputs VW·(4g + x) + e of every 16·VW.
template <int HD, class T>
struct PagedAcc {
    typedef PagedTile<HD, T> Tile;
    static constexpr uint32_t VW = Tile::VW, VN = Tile::VN;
    // weights are 2^BIAS·e^(s − m); m follows the maximum when that has grown by 2^GROW.  f32 pages: so that the
    // largest weight is 1, and a product with the type's largest value finite
    static constexpr float GROW = 3.0f, BIAS = sizeof(T) == 2 ? 15.0f - GROW : -GROW;
    f32x4 o[VN][VW];
    float m, l;
    RT_DEV void start() {
#pragma unroll
        for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
            for (uint32_t e = 0; e < VW; ++e) o[i][e] = f32x4{0, 0, 0, 0};
        m = -__builtin_huge_valf();
        l = 0.0f;
    }
    // products (NEG: unseen), scores in units of log 2 divided by scale, a power of two, to weights.  A column that
    // has seen nothing has the sum 0; the maximum does not tell: it passes NaN over.
    template <uint32_t N>
    RT_DEV void weigh(float (&p)[N], float scale) {
        const float NEG = -__builtin_huge_valf();
        float tmax = p[0];
#pragma unroll
        for (uint32_t r = 1; r < N; ++r) tmax = fmaxf(tmax, p[r]);
        tmax = column_max(tmax) * scale;
        if (__ballot(tmax > m + GROW)) {
            const float mn = fmaxf(m, tmax), md = mn == NEG ? 0.0f : mn, f = __builtin_amdgcn_exp2f(m - md);
            m = mn;
            l *= f;
#pragma unroll
            for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
                for (uint32_t e = 0; e < VW; ++e) o[i][e] *= f;
        }
        const float md = (m == NEG ? 0.0f : m) - BIAS;
#pragma unroll
        for (uint32_t r = 0; r < N; ++r) {
            p[r] = __builtin_amdgcn_exp2f(fmaf(p[r], scale, -md));
            l += p[r];
        }
    }
    RT_DEV void join() {  // the sum over the four lanes of a column
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
    }
    RT_DEV bool finite() const {
        bool bad = !(l < __builtin_huge_valf());
#pragma unroll
        for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
            for (uint32_t e = 0; e < VW; ++e)
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) bad |= !(fabsf(o[i][e][x]) < __builtin_huge_valf());
        return !__ballot(bad);
    }
};

// (a product that no later sum takes in unrounded)
RT_DEV float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

// The tiles t0, t0 + step, ... of a chunk (RUN 2: pairs of tiles there) for 16
// columns on the f32 matrix cores: q is the lane's column, [0, lim) what it sees, limn / limx the
// smallest and largest lim of the columns.
template <int HD, class T, uint32_t RUN = 1>
RT_DEV void paged_f32(PagedAcc<HD, T>& acc, const PagedView<T>& v, const float* q, float scale2, uint32_t t0,
                      uint32_t step, uint32_t lim, uint32_t limn, uint32_t limx) {
    typedef PagedTile<HD, T> Tile;
    constexpr uint32_t KW = Tile::KW, KN = Tile::KN, VW = Tile::VW, VN = Tile::VN;
    const uint32_t lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    auto after = [&](uint32_t t) { return RUN == 2 && t % 2 == 0 ? t + 1 : t + step - (RUN - 1); };
    // the next tile's keys are on their way while this one's weights are made,
    // its values from the second product on
    Tile kv;
    uint32_t page = v.page(t0);
    if (page < v.num_pages) {
        kv.load_k(v.k + v.place(t0, page, HD), lane);
        kv.load_v(v.v + v.place(t0, page, HD), lane);
    }
    float qf[KN][KW];
#pragma unroll
    for (uint32_t i = 0; i < KN; ++i)
#pragma unroll
        for (uint32_t e = 0; e < KW; e += 4) *(f32x4*)&qf[i][e] = *(const f32x4*)(q + i * 4 * KW + g * KW + e);
    acc.start();
    uint32_t next = v.page(after(t0));
    for (uint32_t t = t0; t < v.t1; t = after(t)) {
        const uint32_t p0 = (v.tb + t) * RT_PAGED_TILE, tn = after(t);
        const bool there = page < v.num_pages, more = next < v.num_pages;
        const size_t off = v.place(t, there ? page : 0, HD), offn = v.place(tn, more ? next : 0, HD);
        page = next;
        next = v.page(after(tn));
        f32x4 sa = {0, 0, 0, 0}, sb = {0, 0, 0, 0};
        if (there) {
#pragma unroll
            for (uint32_t i = 0; i < KN; ++i)
#pragma unroll
                for (uint32_t e = 0; e < KW; e += 2) {
                    sa = mfma4((float)kv.k[i][e], qf[i][e], sa);
                    sb = mfma4((float)kv.k[i][e + 1], qf[i][e + 1], sb);
                }
        }
        if (more) kv.load_k(v.k + offn, lane);
        if (there) {
        const bool edge = p0 < v.lo || p0 + RT_PAGED_TILE > limn;
        float p[4];
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            const uint32_t pos = p0 + 4 * g + r;
            p[r] = edge && (pos < v.lo || pos >= lim) ? -__builtin_huge_valf() : rounded_product(sa[r] + sb[r], scale2);
        }
        acc.weigh(p, 1.0f);
        bool bad = false;
        if (edge) {
            // what only later columns see must not reach the earlier ones as 0·∞
            kv.clear(p0 + 4 * g, v.lo, limx);
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
#pragma unroll
                for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
                    for (uint32_t e = 0; e < VW; ++e) bad |= !(fabsf((float)kv.v[r][i][e]) < __builtin_huge_valf());
        }
        if (!__ballot(bad)) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
#pragma unroll
                for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
                    for (uint32_t e = 0; e < VW; ++e) acc.o[i][e] = mfma4((float)kv.v[r][i][e], p[r], acc.o[i][e]);
        } else {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
#pragma unroll 1
                for (uint32_t h = 0; h < 4; ++h) {
                    const float pp = __shfl(p[r], h * 16 + c, 64);
                    const uint32_t pos = p0 + 4 * h + r;
                    if (pos < v.lo || pos >= lim) continue;
                    const T* vp = v.v + off + (size_t)(4 * h + r) * HD + 4 * g * VW;
#pragma unroll
                    for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
                        for (uint32_t e = 0; e < VW; ++e)
#pragma unroll
                            for (uint32_t x = 0; x < 4; ++x)
                                acc.o[i][e][x] = fmaf(pp, (float)vp[i * 16 * VW + x * VW + e], acc.o[i][e][x]);
                }
        }
        }
        if (more) kv.load_v(v.v + offn, lane);
    }
    acc.join();
}

// A column's scaled query as pairs of f16, x·2^e = hi + lo, from the lane's part of it
// and the column's largest; returns 2^-e.
template <uint32_t N>
RT_DEV float split_query(const float (&x)[N][8], float mx, h8_t (&qh)[N], h8_t (&ql)[N]) {
    // (at most 126: 2^-e stays a normal number)
    const int e = mx > 0.0f ? min(126, 15 - __builtin_amdgcn_frexp_expf(mx)) : 0;
    const float f = ldexpf(1.0f, e);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            const float y = x[i][k] * f;
            qh[i][k] = (_Float16)y;
            ql[i][k] = (_Float16)(y - (float)qh[i][k]);
        }
    return ldexpf(1.0f, -e);
}
template <int HD>
RT_DEV float paged_query(const float* q, float scale2, h8_t (&qh)[HD / 32], h8_t (&ql)[HD / 32]) {
    const uint32_t g = (threadIdx.x & 63) >> 4;
    float x[HD / 32][8], mx = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < HD / 32; ++i)
#pragma unroll
        for (uint32_t k = 0; k < 8; k += 4) {
            const f32x4 v = *(const f32x4*)(q + 32 * i + 8 * g + k) * scale2;
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) {
                x[i][k + e] = v[e];
                mx = fmaxf(mx, fabsf(v[e]));
            }
        }
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    return split_query<HD / 32>(x, mx, qh, ql);
}
// (hi towards zero, two at a time; what is left has at most 14 bits, lo the
// nearest of it)
RT_DEV void split_weights(const float* p, h8_t& hi, h8_t& lo) {
    float minus = -1.0f;  // (known, it would be two conversions and subtractions; so it is one mixed fma each)
    asm("" : "+s"(minus));
    typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
    typedef float f2_t __attribute__((ext_vector_type(2)));
#pragma unroll
    for (uint32_t r = 0; r < 8; r += 2) {
        const h2_t h = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_pkrtz(p[r], p[r + 1]));
        const h2_t l = __builtin_convertvector((f2_t{fmaf((float)h[0], minus, p[r]), fmaf((float)h[1], minus, p[r + 1])}), h2_t);
        hi[r] = h[0], hi[r + 1] = h[1];
        lo[r] = l[0], lo[r + 1] = l[1];
    }
}

// The same for f16 pages on the f16 matrix cores, two tiles at a time: t0, t0 +
// 1, t0 + step, ...
template <int HD>
RT_DEV void paged_f16(PagedAcc<HD, _Float16>& acc, const PagedView<_Float16>& v, const float* q, float scale2,
                      uint32_t t0, uint32_t step, uint32_t lim, uint32_t limn, uint32_t limx) {
    typedef PagedTile<HD, _Float16> Tile;
    constexpr uint32_t KN = Tile::KN, VW = Tile::VW, VN = Tile::VN;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4;
    Tile kv[2];
    uint32_t page[2] = {v.page(t0), v.page(t0 + 1)};
    auto keys = [&](const bool (&there)[2], const size_t (&off)[2]) {
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
            if (there[u]) kv[u].load_k(v.k + off[u], lane);
            else kv[u].no_k();
        }
    };
    auto values = [&](const bool (&there)[2], const size_t (&off)[2]) {
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
            if (there[u]) kv[u].load_v(v.v + off[u], lane);
            else kv[u].no_v();
        }
    };
    bool there[2] = {page[0] < v.num_pages, page[1] < v.num_pages};
    {
        const size_t off[2] = {v.place(t0, there[0] ? page[0] : 0, HD), v.place(t0 + 1, there[1] ? page[1] : 0, HD)};
        keys(there, off);
        values(there, off);
    }
    page[0] = v.page(t0 + step), page[1] = v.page(t0 + step + 1);
    h8_t qh[KN], ql[KN];
    const float qs = paged_query<HD>(q, scale2, qh, ql);
    acc.start();
    for (uint32_t t = t0; t < v.t1; t += step) {
        const uint32_t p0 = (v.tb + t) * RT_PAGED_TILE, tn = t + step;
        const bool more[2] = {page[0] < v.num_pages, page[1] < v.num_pages};
        const size_t off[2] = {v.place(tn, more[0] ? page[0] : 0, HD), v.place(tn + 1, more[1] ? page[1] : 0, HD)};
        page[0] = v.page(tn + step), page[1] = v.page(tn + step + 1);
        float p[8];
        const bool edge = p0 < v.lo || p0 + 2 * RT_PAGED_TILE > limn || !there[0] || !there[1];
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
            f32x4 sa = {0, 0, 0, 0}, sb = {0, 0, 0, 0};
#pragma unroll
            for (uint32_t i = 0; i < KN; ++i) {
                sa = mfma32(kv[u].k[i], qh[i], sa);
                sb = mfma32(kv[u].k[i], ql[i], sb);
            }
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) p[4 * u + r] = sa[r] + sb[r];
        }
        keys(more, off);
        if (edge) {
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) {
                const uint32_t pos = p0 + 16 * (r / 4) + 4 * g + r % 4;
                if (pos < v.lo || pos >= lim || !there[r / 4]) p[r] = -__builtin_huge_valf();
            }
            kv[0].clear(p0 + 4 * g, v.lo, limx);
            kv[1].clear(p0 + 16 + 4 * g, v.lo, limx);
        }
        acc.weigh(p, qs);
        h8_t ph, pl;
        split_weights(p, ph, pl);
#pragma unroll
        for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
            for (uint32_t e = 0; e < VW; ++e) {
                h8_t a;
#pragma unroll
                for (uint32_t r = 0; r < 8; ++r) a[r] = kv[r / 4].v[r % 4][i][e];
                acc.o[i][e] = mfma32(a, ph, acc.o[i][e]);
                acc.o[i][e] = mfma32(a, pl, acc.o[i][e]);
            }
        values(more, off);
        there[0] = more[0], there[1] = more[1];
    }
    acc.join();
}

// What a job's workgroup knows of its columns.
template <int HD, class T>
struct PagedCols {
    const PagedAttnArgs& a;
    PagedView<T> v;
    uint32_t kvh, G, row0, col0, ncl, hi;
    bool pre;
    uint32_t rows, kv;  // of the sequence (not pre)
    RT_DEV uint32_t row(uint32_t cc) const { return row0 + (col0 + cc) / G; }
    RT_DEV uint32_t head(uint32_t cc) const { return kvh * G + (col0 + cc) % G; }
    RT_DEV const float* q(uint32_t cc) const { return a.q + ((size_t)row(cc) * a.H + head(cc)) * HD; }
    // positions below it are what a column sees; every lane of the wave calls it
    RT_DEV uint32_t lim(uint32_t cc) const {
        uint32_t back = rows - (col0 + cc) / G, len = kv;  // the row is its sequence's back-th from the end
        if (pre) {
            const PagedBatch& b = a.b;
            const uint32_t r = row(cc);
            uint32_t s = r;
            if (b.row_start) {  // the sequences that end at or before the row
                s = 0;
                for (uint32_t s0 = 0; s0 < b.n_seqs; s0 += 64) {
                    const uint32_t n = min(64u, b.n_seqs - s0), e = b.row_start[s0 + min(threadIdx.x & 63, n - 1) + 1];
                    for (uint32_t x = 0; x < n; ++x) s += (uint32_t)__builtin_amdgcn_readlane(e, x) <= r;
                }
                s = min(s, b.n_seqs - 1);
            }
            const SeqRows sr = seq_rows(b, s);
            back = sr.n - (r - sr.first);
            len = b.kv_len[s];
        }
        return back <= len ? min(len - back + 1, hi) : 0u;
    }
    // where a column's outputs of a chunk go, whole or in part
    template <uint32_t SR>
    RT_DEV float* place(uint32_t job, uint32_t cc, bool alone) const {
        return alone ? a.out + ((size_t)row(cc) * a.H + head(cc)) * HD
                     : a.part + (((size_t)job * a.b.KVH + kvh) * SR + cc) * HD;
    }
    template <uint32_t SR>
    RT_DEV void state(const PagedJob& j, uint32_t job, uint32_t cc, float m, float l, bool alone) const {
        const size_t slot = ((size_t)job * a.b.KVH + kvh) * SR + cc;
        if (!alone) {
            a.ml[2 * slot] = m;
            a.ml[2 * slot + 1] = l;
        }
        if (j.chunk == 0) note<SR>(j, (size_t)row(cc) * a.H + head(cc), cc);
    }
    // of 16 columns
    template <uint32_t SR>
    RT_DEV void put(const PagedAcc<HD, T>& acc, const PagedJob& j, uint32_t job, uint32_t cc, bool alone) const {
        constexpr uint32_t VW = PagedTile<HD, T>::VW, VN = PagedTile<HD, T>::VN;
        if (cc >= ncl) return;
        const uint32_t g = (threadIdx.x & 63) >> 4;
        float* o = place<SR>(job, cc, alone);
        const float f = !alone ? 1.0f : acc.l == 0.0f ? 0.0f : 1.0f / acc.l;
#pragma unroll
        for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
            for (uint32_t x = 0; x < 4; ++x)
#pragma unroll
                for (uint32_t e = 0; e < VW; e += 4) {
                    f32x4 y;
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) y[k] = acc.o[i][e + k][x] * f;
                    *(f32x4*)(o + i * 16 * VW + (4 * g + x) * VW + e) = y;
                }
        if (g == 0) state<SR>(j, job, cc, acc.m, acc.l, alone);
    }
    template <uint32_t SR>
    RT_DEV void note(const PagedJob& j, size_t rh, uint32_t cc) const {
        uint32_t* in = a.info + (rh * 2 + (pre ? 1 : 0)) * 2;
        in[0] = j.first;
        in[1] = j.chunks * SR + cc;
    }
};

template <int HD, class T, bool WIDE>
RT_DEV void paged_narrow(const PagedAttnArgs& a, const PagedCols<HD, T>& co, const PagedJob& j, uint32_t job,
                         float* lds) {
    constexpr uint32_t NW = RT_PAGED_WAVES, SR = paged_slot_rows<WIDE>();
    constexpr uint32_t VW = PagedTile<HD, T>::VW, VN = PagedTile<HD, T>::VN;
    float (*olds)[16][HD + 4] = (float (*)[16][HD + 4])lds;
    float (*mlds)[16] = (float (*)[16])(lds + NW * 16 * (HD + 4)), (*llds)[16] = mlds + NW;
    const PagedBatch& b = a.b;
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t c = lane & 15, g = lane >> 4, ncl = co.ncl, cc = min(c, ncl - 1), lim = co.lim(cc);
    uint32_t limx = lim, limn = lim;  // of the block's columns: the largest, the smallest
    for (uint32_t o = 1; o < 16; o *= 2) {
        limx = max(limx, __shfl_xor(limx, o, 64));
        limn = min(limn, __shfl_xor(limn, o, 64));
    }
    limx = __builtin_amdgcn_readfirstlane(limx);
    limn = __builtin_amdgcn_readfirstlane(limn);
    PagedView<T> v = co.v;
    v.t1 = min(v.t1, limx > v.lo ? (limx + RT_PAGED_TILE - 1) / RT_PAGED_TILE - v.tb : 0u);
    const float NEG = -__builtin_huge_valf(), scale2 = a.scale * 1.44269504f;
    const uint32_t t0 = j.chunk * NW + w, stride = j.chunks * NW;
    PagedAcc<HD, T> acc;
    if constexpr (sizeof(T) == 2) {
        paged_f16<HD>(acc, v, co.q(cc), scale2, 2 * t0, 2 * stride, lim, limn, limx);
        if (!acc.finite()) paged_f32<HD, T, 2>(acc, v, co.q(cc), scale2, 2 * t0, 2 * stride, lim, limn, limx);
    } else {
        paged_f32<HD, T>(acc, v, co.q(cc), scale2, t0, stride, lim, limn, limx);
    }
#pragma unroll
    for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x)
#pragma unroll
            for (uint32_t e = 0; e < VW; ++e) olds[w][c][i * 16 * VW + (4 * g + x) * VW + e] = acc.o[i][e][x];
    if (g == 0) {
        mlds[w][c] = acc.m;
        llds[w][c] = acc.l;
    }
    __syncthreads();
    const bool noted = WIDE || a.shared_len, alone = j.chunks == 1 && !a.shared_len;
    for (uint32_t i = tid; i < 16 * HD / 4; i += 64 * NW) {
        const uint32_t k = i / (HD / 4), d = i % (HD / 4) * 4;
        if (k >= ncl) break;
        float M = mlds[0][k];
#pragma unroll
        for (uint32_t u = 1; u < NW; ++u) M = fmaxf(M, mlds[u][k]);
        const float md = M == NEG ? 0.0f : M;
        f32x4 o = {0, 0, 0, 0};
        float L = 0.0f;
#pragma unroll
        for (uint32_t u = 0; u < NW; ++u) {
            // (one that the others outweigh keeps its NaN, one that saw nothing adds nothing)
            const float f = mlds[u][k] == NEG ? 0.0f : __builtin_amdgcn_exp2f(mlds[u][k] - md);
            L += f * llds[u][k];
            o += f * *(const f32x4*)&olds[u][k][d];
        }
        const size_t slot = ((size_t)job * b.KVH + co.kvh) * SR + k, rh = (size_t)co.row(k) * a.H + co.head(k);
        if (alone) {
            *(f32x4*)(a.out + rh * HD + d) = L == 0.0f ? f32x4{0, 0, 0, 0} : o / L;
        } else if (noted) {
            *(f32x4*)(a.part + slot * HD + d) = o;
            if (d == 0) {
                a.ml[2 * slot] = M;
                a.ml[2 * slot + 1] = L;
            }
        } else {
#pragma unroll
            for (uint32_t x = 0; x < 4; x += 2) dev_store((uint64_t*)(a.part + slot * HD + d + x), pair_of(o[x], o[x + 1]));
            if (d == 0) dev_store((uint64_t*)(a.ml + 2 * slot), pair_of(M, L));
        }
        if (noted && d == 0 && j.chunk == 0) co.template note<SR>(j, rh, k);
    }
    if (alone || noted) return;
    // The block's last workgroup to arrive puts its chunks together; of more
    // than 24, the last of each group of about √chunks those of the group first.
    // All loads of sixteen chunks are in flight at once.
    __shared__ uint32_t turn;
    constexpr uint32_t PW = HD / 2, PT = 16 * PW / (64 * NW), BATCH = 16;  // pairs a row, a thread; chunks at a time
    __shared__ float mc[BATCH][16], lc[BATCH][16];
    auto last_of = [&](uint32_t* counter, uint32_t n) {
        dev_stores_done();
        __syncthreads();
        if (tid == 0) {
            turn = arrive(counter);
            if (turn == n - 1) dev_store(counter, 0u);
        }
        __syncthreads();
        return turn == n - 1;
    };
    auto slot_of = [&](uint32_t jb) { return ((size_t)jb * b.KVH + co.kvh) * SR; };
    // jobs at, at + step, ... (n of them): into the outputs, or the first one's place
    auto meet = [&](uint32_t at, uint32_t step, uint32_t n, bool out) {
        const uint32_t items = ncl * PW;
        float o[PT][2], L[PT], M[PT];
#pragma unroll
        for (uint32_t u = 0; u < PT; ++u) o[u][0] = o[u][1] = L[u] = 0.0f, M[u] = NEG;
        for (uint32_t x0 = 0; x0 < n; x0 += BATCH) {
            uint64_t x[PT][BATCH];
            const uint32_t mk = tid & 15, my = tid >> 4;
            uint64_t ml = pair_of(NEG, 0.0f);
            if (x0 + my < n && mk < ncl) ml = dev_load((const uint64_t*)a.ml + slot_of(at + (x0 + my) * step) + mk);
#pragma unroll
            for (uint32_t u = 0; u < PT; ++u)
                if (256 * u < items) {
                    const uint32_t i = min(tid + 256 * u, items - 1);
#pragma unroll
                    for (uint32_t y = 0; y < BATCH; ++y)
                        if (x0 + y < n) x[u][y] = dev_load((const uint64_t*)(a.part + slot_of(at + (x0 + y) * step) * HD) + i);
                }
            if (x0) __syncthreads();
            mc[my][mk] = pair_lo(ml);
            lc[my][mk] = pair_hi(ml);
            __syncthreads();
#pragma unroll
            for (uint32_t u = 0; u < PT; ++u)
                if (256 * u < items) {
                    const uint32_t k = min(tid + 256 * u, items - 1) / PW;
                    float mx = M[u];
#pragma unroll
                    for (uint32_t y = 0; y < BATCH; ++y) mx = fmaxf(mx, mc[y][k]);
                    const float md = mx == NEG ? 0.0f : mx, f0 = __builtin_amdgcn_exp2f(M[u] - md);
                    o[u][0] *= f0, o[u][1] *= f0, L[u] *= f0;
                    M[u] = mx;
#pragma unroll
                    for (uint32_t y = 0; y < BATCH; ++y)
                        if (x0 + y < n) {
                            const bool none = mc[y][k] == NEG;  // (its sums are zeros)
                            const float f = none ? 0.0f : __builtin_amdgcn_exp2f(mc[y][k] - md);
                            L[u] = fmaf(f, lc[y][k], L[u]);
                            o[u][0] = fmaf(f, pair_lo(x[u][y]), o[u][0]);
                            o[u][1] = fmaf(f, pair_hi(x[u][y]), o[u][1]);
                        }
                }
        }
        if (!out) __syncthreads();  // (all have read the place that is written now)
#pragma unroll
        for (uint32_t u = 0; u < PT; ++u) {
            const uint32_t i = tid + 256 * u, k = i / PW, d = i % PW * 2;
            if (i >= items) break;
            if (out) {
                float* op = a.out + ((size_t)co.row(k) * a.H + co.head(k)) * HD + d;
                op[0] = L[u] == 0.0f ? 0.0f : o[u][0] / L[u];
                op[1] = L[u] == 0.0f ? 0.0f : o[u][1] / L[u];
            } else {
                const size_t slot = slot_of(at) + k;
                dev_store((uint64_t*)(a.part + slot * HD + d), pair_of(o[u][0], o[u][1]));
                if (d == 0) dev_store((uint64_t*)(a.ml + 2 * slot), pair_of(M[u], L[u]));
            }
        }
    };
    uint32_t* whole = a.counters + 2 * (j.first * b.KVH + co.kvh);
    uint32_t step = 1, n = j.chunks;
    if (n > 24) {
        step = (uint32_t)ceilf(sqrtf((float)n));
        const uint32_t grp = j.chunk / step, gn = min(step, n - grp * step), at = j.first + grp * step;
        if (gn > 1) {
            if (!last_of(a.counters + 2 * (at * b.KVH + co.kvh) + 1, gn)) return;
            meet(at, 1, gn, false);
        }
        n = (n + step - 1) / step;
    }
    if (last_of(whole, n)) meet(j.first, step, n, true);
}

// Stages of two tiles in LDS, brought three ahead, nothing through registers: 32
// rows of keys, 32 of values, as they are but for their 16-byte pieces, permuted
// by the row so that the reads (keys: 16 rows' same piece; values, transposing:
// four pieces of eight rows) meet all banks.
template <int HD>
struct PagedStage {
    static constexpr uint32_t ROW = HD / 8, LEN = 64 * ROW, N = 4;  // in 16 bytes
    static constexpr uint32_t LOADS = LEN / 64 / RT_PAGED_WAVES;    // of a wave
    // place of piece p of row r (32 ..: values)
    static RT_DEV uint32_t piece(uint32_t r, uint32_t p) {
        const uint32_t x = r < 32 ? (HD == 64 ? r >> 1 & 7 : r & 15) : (HD == 64 ? r << 1 & 4 : r << 2 & 12);
        return r * ROW + (p ^ x);
    }
};
// 16 bytes a lane from p (the lane's own) to LDS, lane 0's at byte `at`, each
// next behind it.  No registers receive it, and the compiler knows nothing of
// it: with the builtin it would wait for all of them at each read of LDS.
// stages_left() is the wait.
RT_DEV void bring16(const void* p, uint32_t at) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(at) : "memory", "m0");
}
// waits until at most n of the wave's stages are on their way
template <uint32_t LOADS>
RT_DEV void stages_left(uint32_t n) {
    constexpr auto wait = [](uint32_t c) constexpr { return (c & 15) | (c >> 4) << 14 | 7 << 4 | 15 << 8; };
    if (n >= 2) __builtin_amdgcn_s_waitcnt(wait(2 * LOADS));
    else if (n == 1) __builtin_amdgcn_s_waitcnt(wait(LOADS));
    else __builtin_amdgcn_s_waitcnt(wait(0));
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

template <int HD, class T, bool WIDE>
RT_DEV void paged_attn(const PagedAttnArgs& a) {
    constexpr uint32_t NARROW = RT_PAGED_WAVES * 16 * (HD + 4 + 2) / 4;  // in 16 bytes
    constexpr uint32_t STAGES = WIDE ? PagedStage<HD>::N * PagedStage<HD>::LEN : 0;
    __shared__ f32x4 lds[NARROW > STAGES ? NARROW : STAGES];
    const PagedBatch& b = a.b;
    const uint32_t kvh = blockIdx.x % b.KVH, job = blockIdx.x / b.KVH;
    const PagedJob j = paged_job<HD, T, WIDE>(a, job);
    // (row starts that are not in order may plan more jobs than the launch has)
    if (!j.any || j.chunks > a.jobs - j.first) return;
    const uint32_t G = a.H / b.KVH, cap = b.table_stride << b.ps_shift;
    const bool pre = j.seq == b.n_seqs;
    const uint32_t rows = j.rows, lo = pre ? 0 : a.shared_len, hi = min(j.kv, cap);
    const uint32_t* table = pre ? a.shared_table : b.table + (size_t)j.seq * b.table_stride;
    const uint32_t bc = paged_block<WIDE>(rows * G), col0 = j.rb * bc;
    const size_t head = ((size_t)kvh << b.ps_shift) * HD;
    const uint32_t tb = lo / RT_PAGED_TILE, tend = hi > lo ? (hi + RT_PAGED_TILE - 1) / RT_PAGED_TILE - tb : 0;
    const PagedView<T> v{(const T*)b.k + head, (const T*)b.v + head, table, b.page_stride, b.num_pages, b.ps_shift,
                         tb, tend, lo};
    const PagedCols<HD, T> co{a, v, kvh, G, j.row0, col0, min(bc, rows * G - col0), hi, pre, rows, j.kv};
    if constexpr (WIDE) {
        if (bc > RT_PAGED_ROWS) {
            paged_wide<HD>(a, co, j, job, (h8_t*)lds);
            return;
        }
    }
    paged_narrow<HD, T, WIDE>(a, co, j, job, (float*)lds);
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
