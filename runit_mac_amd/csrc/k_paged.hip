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
// 2^-24 of itself, half a percent of a radian at position 100,000.
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
// — are taken in blocks of 16 columns of the f32 matrix cores, and its
// positions in tiles of 16.  A job is a block over a chunk of tiles, one
// workgroup; its four waves take every fourth tile, each with a softmax of its
// own, and meet in LDS.  Chunks meet in k_paged_merge.

// The jobs of one KV head: blocks × chunks of every sequence in turn (and, with
// a shared prefix, before them those of all rows over it).  The chunk length
// comes from the work that the device finds, so that the jobs are alike
// whatever the lengths: jobs ≤ blocks + target.
struct PagedJob {
    uint32_t seq;             // n_seqs: the shared prefix
    uint32_t rb, chunk, first, chunks;  // block, chunk, first job of the block, its chunks
    uint32_t tile0, len;      // first tile of the chunk, tiles of a chunk
    bool any;
};
RT_DEV uint32_t paged_tiles(const PagedAttnArgs& a, uint32_t s) {  // a sequence's own tiles
    const uint32_t cap = a.b.table_stride << a.b.ps_shift, L = min(a.b.kv_len[s], cap);
    const uint32_t t0 = a.shared_len / RT_PAGED_TILE;
    const uint32_t t1 = (L + RT_PAGED_TILE - 1) / RT_PAGED_TILE;
    return L > a.shared_len ? t1 - t0 : 0;
}
RT_DEV uint32_t wave_scan_add(uint32_t v) {  // inclusive
    const uint32_t lane = threadIdx.x & 63;
    for (uint32_t o = 1; o < 64; o *= 2) {
        const uint32_t u = __shfl_up(v, o, 64);
        v += lane >= o ? u : 0;
    }
    return v;
}
RT_DEV PagedJob paged_job(const PagedAttnArgs& a, uint32_t job) {
    const uint32_t lane = threadIdx.x & 63, G = a.H / a.b.KVH, n = a.b.n_seqs;
    const uint32_t rows = a.b.row_start ? min(a.b.row_start[n], a.b.rows) : min(n, a.b.rows);
    const uint32_t pb = a.shared_len ? (rows * G + RT_PAGED_ROWS - 1) / RT_PAGED_ROWS : 0;
    const uint32_t pt = (a.shared_len + RT_PAGED_TILE - 1) / RT_PAGED_TILE;
    // (tiles × blocks of 2^28 positions in all: below 2^64)
    uint64_t work = 0;
    for (uint32_t s = lane; s < n; s += 64)
        work += (uint64_t)((seq_rows(a.b, s).n * G + RT_PAGED_ROWS - 1) / RT_PAGED_ROWS) * paged_tiles(a, s);
    for (uint32_t o = 32; o; o /= 2) work += __shfl_xor((unsigned long long)work, o, 64);
    work += (uint64_t)pb * pt;
    PagedJob j{};
    uint64_t len = a.target ? (work + a.target - 1) / a.target : 0x7fffffffu;
    len = max((uint64_t)a.min_chunk, (len + RT_PAGED_WAVES - 1) / RT_PAGED_WAVES * RT_PAGED_WAVES);
    j.len = (uint32_t)min(len, (uint64_t)0x7ffffffc);
    auto chunks = [&](uint32_t tiles) { return max(1u, tiles / j.len + (tiles % j.len ? 1u : 0u)); };
    auto found = [&](uint32_t seq, uint32_t base, uint32_t nc) {
        const uint32_t k = job - base;
        j.seq = seq;
        j.rb = k / nc;
        j.chunk = k % nc;
        j.first = job - j.chunk;
        j.chunks = nc;
        j.tile0 = j.chunk * j.len;
        j.any = true;
    };
    uint32_t base = 0;
    if (pb) {
        const uint32_t nc = chunks(pt);
        if (job < pb * nc) {
            found(n, 0, nc);
            return j;
        }
        base = pb * nc;
    }
    for (uint32_t s0 = 0; s0 < n; s0 += 64) {
        const uint32_t s = s0 + lane;
        uint32_t mine = 0, nc = 1;
        if (s < n) {
            nc = chunks(paged_tiles(a, s));
            mine = (seq_rows(a.b, s).n * G + RT_PAGED_ROWS - 1) / RT_PAGED_ROWS * nc;
        }
        const uint32_t upto = base + wave_scan_add(mine);
        const uint64_t hit = __ballot(job < upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            found(s0 + l, __shfl(upto - mine, l, 64), __shfl(nc, l, 64));
            return j;
        }
        base = __shfl(upto, 63, 64);
    }
    return j;
}

// Operands of a tile.  Keys: lane l holds position l % 16, W of every 4W
// elements from W·(l / 16) on; values: of the positions 4(l / 16) + t, W of
// every 16W elements from W·(l % 16) on.
template <int HD, class T>
struct PagedTile {
    static constexpr uint32_t KW = sizeof(T) == 4 ? 4 : 8, KN = HD / (4 * KW);
    static constexpr uint32_t VW = sizeof(T) == 4 || HD == 64 ? 4 : 8, VN = HD / (16 * VW);
    typedef T kvec __attribute__((ext_vector_type(KW)));
    typedef T vvec __attribute__((ext_vector_type(VW)));
    kvec k[KN];
    vvec v[4][VN];
    RT_DEV void load(const T* kb, const T* vb, uint32_t lane) {
        const T* kp = kb + (size_t)(lane & 15) * HD + (lane >> 4) * KW;
#pragma unroll
        for (uint32_t i = 0; i < KN; ++i) k[i] = *(const kvec*)(kp + i * 4 * KW);
#pragma unroll
        for (uint32_t t = 0; t < 4; ++t) {
            const T* vp = vb + (size_t)(4 * (lane >> 4) + t) * HD + (lane & 15) * VW;
#pragma unroll
            for (uint32_t i = 0; i < VN; ++i) v[t][i] = *(const vvec*)(vp + i * 16 * VW);
        }
    }
};

RT_DEV uint64_t pair_of(float lo, float hi) {
    return (uint64_t)__builtin_bit_cast(uint32_t, hi) << 32 | __builtin_bit_cast(uint32_t, lo);
}
RT_DEV float pair_lo(uint64_t p) { return __builtin_bit_cast(float, (uint32_t)p); }
RT_DEV float pair_hi(uint64_t p) { return __builtin_bit_cast(float, (uint32_t)(p >> 32)); }

template <int HD, class T>
RT_DEV void paged_attn(const PagedAttnArgs& a) {
    typedef PagedTile<HD, T> Tile;
    constexpr uint32_t KW = Tile::KW, KN = Tile::KN, VW = Tile::VW, VN = Tile::VN, NW = RT_PAGED_WAVES;
    __shared__ float olds[NW][16][HD + 4];
    __shared__ float mlds[NW][16], llds[NW][16];
    const PagedBatch& b = a.b;
    const uint32_t tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t c = lane & 15, g = lane >> 4, kvh = blockIdx.x % b.KVH, job = blockIdx.x / b.KVH;
    const PagedJob j = paged_job(a, job);
    if (!j.any) return;
    const uint32_t G = a.H / b.KVH, cap = b.table_stride << b.ps_shift;
    const bool pre = j.seq == b.n_seqs;
    // a column's row, head, and the positions it sees: [lo, lim)
    uint32_t ncol, row0, lo, hi;
    const uint32_t* table;
    if (pre) {
        row0 = 0;
        ncol = (b.row_start ? min(b.row_start[b.n_seqs], b.rows) : min(b.n_seqs, b.rows)) * G;
        lo = 0;
        hi = a.shared_len;
        table = a.shared_table;
    } else {
        const SeqRows sr = seq_rows(b, j.seq);
        row0 = sr.first;
        ncol = sr.n * G;
        lo = a.shared_len;
        hi = min(b.kv_len[j.seq], cap);
        table = b.table + (size_t)j.seq * b.table_stride;
    }
    const uint32_t col0 = j.rb * RT_PAGED_ROWS, ncl = min(RT_PAGED_ROWS, ncol - col0);  // columns of the block
    auto row_of = [&](uint32_t cc) { return row0 + (col0 + cc) / G; };
    auto lim_of = [&](uint32_t cc) {
        const uint32_t row = row_of(cc);
        uint32_t s = j.seq;
        if (pre) {  // the row's sequence
            if (!b.row_start) {
                s = row;
            } else {
                uint32_t x = 0, y = b.n_seqs;
                while (y - x > 1) {
                    const uint32_t mid = (x + y) / 2;
                    if (b.row_start[mid] <= row) x = mid; else y = mid;
                }
                s = x;
            }
        }
        const SeqRows sr = seq_rows(b, s);
        const uint32_t back = sr.n - (row - sr.first), len = b.kv_len[s];
        return back <= len ? min(len - back + 1, hi) : 0u;
    };
    const uint32_t cc = min(c, ncl - 1), head = kvh * G + (col0 + cc) % G;
    const uint32_t lim = lim_of(cc);
    uint32_t limx = lim, limn = lim;  // of the block's rows: the largest, the smallest
    for (uint32_t o = 1; o < 16; o *= 2) {
        limx = max(limx, __shfl_xor(limx, o, 64));
        limn = min(limn, __shfl_xor(limn, o, 64));
    }
    limx = __builtin_amdgcn_readfirstlane(limx);
    limn = __builtin_amdgcn_readfirstlane(limn);
    const uint32_t tb = lo / RT_PAGED_TILE;
    const uint32_t tend = limx > lo ? (limx + RT_PAGED_TILE - 1) / RT_PAGED_TILE - tb : 0;
    const uint32_t t1 = min(tend, j.tile0 + j.len);
    const T* kbase = (const T*)b.k + (((size_t)kvh << b.ps_shift) * HD);
    const T* vbase = (const T*)b.v + (((size_t)kvh << b.ps_shift) * HD);

    float qf[KN][KW];
    const float* qp = a.q + ((size_t)row_of(cc) * a.H + head) * HD;
#pragma unroll
    for (uint32_t i = 0; i < KN; ++i)
#pragma unroll
        for (uint32_t e = 0; e < KW; e += 4)
            *(f32x4*)&qf[i][e] = *(const f32x4*)(qp + i * 4 * KW + g * KW + e);
    f32x4 acc[VN][VW];
#pragma unroll
    for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
        for (uint32_t e = 0; e < VW; ++e) acc[i][e] = f32x4{0, 0, 0, 0};
    const float NEG = -__builtin_huge_valf(), scale2 = a.scale * 1.44269504f;
    float m = NEG, l = 0.0f;  // (in units of log 2)
    // the next tile's operands are loaded while one is computed, its page id
    // before that
    auto entry = [&](uint32_t t) { return t < t1 ? table[(tb + t) * RT_PAGED_TILE >> b.ps_shift] : b.num_pages; };
    auto place = [&](uint32_t t, uint32_t page) {
        return page * b.page_stride + (size_t)((tb + t) * RT_PAGED_TILE & ((1u << b.ps_shift) - 1)) * HD;
    };
    constexpr bool AHEAD = HD < 256;  // (256: two tiles' operands are more registers than there are)
    Tile kv, nx;
    uint32_t page = entry(j.tile0 + w), pnext = entry(j.tile0 + w + NW);
    if (AHEAD && page < b.num_pages) kv.load(kbase + place(j.tile0 + w, page), vbase + place(j.tile0 + w, page), lane);
    for (uint32_t t = j.tile0 + w; t < t1; t += NW) {
        const uint32_t p0 = (tb + t) * RT_PAGED_TILE, pthis = page;
        page = pnext;
        if (AHEAD && page < b.num_pages) nx.load(kbase + place(t + NW, page), vbase + place(t + NW, page), lane);
        if (!AHEAD && pthis < b.num_pages) kv.load(kbase + place(t, pthis), vbase + place(t, pthis), lane);
        pnext = entry(t + 2 * NW);
        if (pthis < b.num_pages) {
        const size_t off = place(t, pthis);
        f32x4 sa = {0, 0, 0, 0}, sb = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t i = 0; i < KN; ++i)
#pragma unroll
            for (uint32_t e = 0; e < KW; e += 2) {
                sa = __builtin_amdgcn_mfma_f32_16x16x4f32((float)kv.k[i][e], qf[i][e], sa, 0, 0, 0);
                sb = __builtin_amdgcn_mfma_f32_16x16x4f32((float)kv.k[i][e + 1], qf[i][e + 1], sb, 0, 0, 0);
            }
        float p[4], tmax = NEG;
        const bool edge = p0 < lo || p0 + RT_PAGED_TILE > limn;
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            p[r] = (sa[r] + sb[r]) * scale2;
            const uint32_t pos = p0 + 4 * g + r;
            if (edge && (pos < lo || pos >= lim)) p[r] = NEG;
            tmax = fmaxf(tmax, p[r]);
        }
        tmax = fmaxf(tmax, __shfl_xor(tmax, 16, 64));
        tmax = fmaxf(tmax, __shfl_xor(tmax, 32, 64));
        const float mn = fmaxf(m, tmax), md = mn == NEG ? 0.0f : mn;
        const float alpha = __builtin_amdgcn_exp2f(m - md);
        m = mn;
        l *= alpha;
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r) {
            p[r] = __builtin_amdgcn_exp2f(p[r] - md);
            l += p[r];
        }
#pragma unroll
        for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
            for (uint32_t e = 0; e < VW; ++e) acc[i][e] *= alpha;
        bool bad = false;
        if (edge) {
            // positions that no row sees may hold anything: zeros; one that only
            // later rows see must not reach the earlier ones as 0·∞
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) {
                const uint32_t pos = p0 + 4 * g + r;
                const bool none = pos < lo || pos >= limx;
#pragma unroll
                for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
                    for (uint32_t e = 0; e < VW; ++e) {
                        if (none) kv.v[r][i][e] = (T)0.0f;
                        bad |= !(fabsf((float)kv.v[r][i][e]) < __builtin_huge_valf());
                    }
            }
        }
        if (!__ballot(bad)) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
#pragma unroll
                for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
                    for (uint32_t e = 0; e < VW; ++e)
                        acc[i][e] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)kv.v[r][i][e], p[r], acc[i][e], 0, 0, 0);
        } else {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r)
#pragma unroll 1
                for (uint32_t h = 0; h < 4; ++h) {
                    const float pp = __shfl(p[r], h * 16 + c, 64);
                    const uint32_t pos = p0 + 4 * h + r;
                    if (pos < lo || pos >= lim) continue;
                    const T* vp = vbase + off + (size_t)(4 * h + r) * HD + 4 * g * VW;
#pragma unroll
                    for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
                        for (uint32_t e = 0; e < VW; ++e)
#pragma unroll
                            for (uint32_t x = 0; x < 4; ++x)
                                acc[i][e][x] = fmaf(pp, (float)vp[i * 16 * VW + x * VW + e], acc[i][e][x]);
                }
        }
        }
        if constexpr (AHEAD) kv = nx;
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // lane (c, g) holds column c's elements VW·(4g + x) + e of every 16·VW
#pragma unroll
    for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
        for (uint32_t x = 0; x < 4; ++x)
#pragma unroll
            for (uint32_t e = 0; e < VW; ++e) olds[w][c][i * 16 * VW + (4 * g + x) * VW + e] = acc[i][e][x];
    if (g == 0) {
        mlds[w][c] = m;
        llds[w][c] = l;
    }
    __syncthreads();
    const bool alone = j.chunks == 1 && !a.shared_len;
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
        const uint32_t row = row_of(k), hd = kvh * G + (col0 + k) % G;
        const size_t slot = ((size_t)job * b.KVH + kvh) * RT_PAGED_ROWS + k;
        if (alone) {
            *(f32x4*)(a.out + ((size_t)row * a.H + hd) * HD + d) = M == NEG ? f32x4{0, 0, 0, 0} : o / L;
        } else if (a.shared_len) {
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
        if (a.shared_len && d == 0 && j.chunk == 0) {
            uint32_t* in = a.info + (((size_t)row * a.H + hd) * 2 + (pre ? 1 : 0)) * 2;
            in[0] = j.first;
            in[1] = j.chunks * 16 + k;
        }
    }
    if (alone || a.shared_len) return;
    // The block's last workgroup to arrive puts its chunks together; of more
    // than 12, the last of each group of about √chunks those of the group first.
    __shared__ uint32_t turn;
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
    auto slot_of = [&](uint32_t jb) { return ((size_t)jb * b.KVH + kvh) * RT_PAGED_ROWS; };
    // jobs at, at + step, ... (n of them), in their order: into the outputs, or the first one's place
    auto meet = [&](uint32_t at, uint32_t step, uint32_t n, bool out) {
        constexpr uint32_t PW = HD / 2, PT = 16 * PW / (64 * NW);  // pairs a row, a thread
        float o[PT][2], L[PT], M[PT];
#pragma unroll
        for (uint32_t u = 0; u < PT; ++u) o[u][0] = o[u][1] = L[u] = 0.0f, M[u] = NEG;
        for (uint32_t x0 = 0; x0 < n; x0 += 8) {
#pragma unroll
            for (uint32_t u = 0; u < PT; ++u) {
                const uint32_t i = tid + u * 64 * NW, k = i / PW, d = i % PW * 2;
                if (k >= ncl) break;
                uint64_t v[8], ml[8];
#pragma unroll
                for (uint32_t x = 0; x < 8; ++x) {
                    const size_t slot = slot_of(at + min(x0 + x, n - 1) * step) + k;
                    ml[x] = dev_load((const uint64_t*)(a.ml + 2 * slot));
                    v[x] = dev_load((const uint64_t*)(a.part + slot * HD + d));
                }
                float mx = M[u];
#pragma unroll
                for (uint32_t x = 0; x < 8; ++x) mx = fmaxf(mx, pair_lo(ml[x]));
                const float md = mx == NEG ? 0.0f : mx, f0 = __builtin_amdgcn_exp2f(M[u] - md);
                o[u][0] *= f0, o[u][1] *= f0, L[u] *= f0;
                M[u] = mx;
#pragma unroll
                for (uint32_t x = 0; x < 8; ++x) {
                    if (x0 + x >= n || pair_lo(ml[x]) == NEG) continue;
                    const float f = __builtin_amdgcn_exp2f(pair_lo(ml[x]) - md);
                    L[u] = fmaf(f, pair_hi(ml[x]), L[u]);
                    o[u][0] = fmaf(f, pair_lo(v[x]), o[u][0]);
                    o[u][1] = fmaf(f, pair_hi(v[x]), o[u][1]);
                }
            }
        }
        if (!out) __syncthreads();  // (all have read the place that is written now)
#pragma unroll
        for (uint32_t u = 0; u < PT; ++u) {
            const uint32_t i = tid + u * 64 * NW, k = i / PW, d = i % PW * 2;
            if (k >= ncl) break;
            if (out) {
                float* op = a.out + ((size_t)row_of(k) * a.H + kvh * G + (col0 + k) % G) * HD + d;
                op[0] = M[u] == NEG ? 0.0f : o[u][0] / L[u];
                op[1] = M[u] == NEG ? 0.0f : o[u][1] / L[u];
            } else {
                const size_t slot = slot_of(at) + k;
                dev_store((uint64_t*)(a.part + slot * HD + d), pair_of(o[u][0], o[u][1]));
                if (d == 0) dev_store((uint64_t*)(a.ml + 2 * slot), pair_of(M[u], L[u]));
            }
        }
    };
    uint32_t* whole = a.counters + 2 * (j.first * b.KVH + kvh);
    uint32_t step = 1, n = j.chunks;
    if (n > 12) {
        step = (uint32_t)ceilf(sqrtf((float)n));
        const uint32_t grp = j.chunk / step, gn = min(step, n - grp * step), at = j.first + grp * step;
        if (gn > 1) {
            if (!last_of(a.counters + 2 * (at * b.KVH + kvh) + 1, gn)) return;
            meet(at, 1, gn, false);
        }
        n = (n + step - 1) / step;
    }
    if (last_of(whole, n)) meet(j.first, step, n, true);
}

// o = Σ o_c·2^(m_c − M) / Σ l_c·2^(m_c − M) over a row's chunks, in their order
template <int HD>
RT_DEV void paged_merge(const PagedAttnArgs& a) {
    constexpr uint32_t TH = HD / 4;
    const PagedBatch& b = a.b;
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, rh = i / TH, d = i % TH * 4;
    const uint32_t rows = b.row_start ? min(b.row_start[b.n_seqs], b.rows) : min(b.n_seqs, b.rows);
    if (rh >= rows * a.H) return;
    const uint32_t kvh = rh % a.H / (a.H / b.KVH);
    const uint32_t* in = a.info + (size_t)rh * 4;
    constexpr uint32_t parts = 2;  // the prefix, the sequence's own positions
    const float NEG = -__builtin_huge_valf();
    float M = NEG;
    for (uint32_t p = 0; p < parts; ++p) {
        const uint32_t first = in[2 * p], n = in[2 * p + 1] / 16, k = in[2 * p + 1] % 16;
        if (first >= a.jobs || n > a.jobs - first) return;
        for (uint32_t u = 0; u < n; ++u)
            M = fmaxf(M, a.ml[2 * (((size_t)(first + u) * b.KVH + kvh) * RT_PAGED_ROWS + k)]);
    }
    const float md = M == NEG ? 0.0f : M;
    float L = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    for (uint32_t p = 0; p < parts; ++p) {
        const uint32_t first = in[2 * p], n = in[2 * p + 1] / 16, k = in[2 * p + 1] % 16;
        for (uint32_t u = 0; u < n; ++u) {
            const size_t slot = ((size_t)(first + u) * b.KVH + kvh) * RT_PAGED_ROWS + k;
            const float mc = a.ml[2 * slot], f = mc == NEG ? 0.0f : __builtin_amdgcn_exp2f(mc - md);
            L += f * a.ml[2 * slot + 1];
            o += f * *(const f32x4*)(a.part + slot * HD + d);
        }
    }
    *(f32x4*)(a.out + (size_t)rh * HD + d) = M == NEG ? f32x4{0, 0, 0, 0} : o / L;
}

#define RT_PAGED_KERNELS(HD)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) k_paged_append_f32_hd##HD(PagedAppendArgs a) {     \
        paged_append<HD, float>(a);                                                                       \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) k_paged_append_f16_hd##HD(PagedAppendArgs a) {     \
        paged_append<HD, _Float16>(a);                                                                    \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256, 2) k_paged_attn_f32_hd##HD(PagedAttnArgs a) {         \
        paged_attn<HD, float>(a);                                                                         \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256, 2) k_paged_attn_f16_hd##HD(PagedAttnArgs a) {         \
        paged_attn<HD, _Float16>(a);                                                                      \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) k_paged_merge_hd##HD(PagedAttnArgs a) {            \
        paged_merge<HD>(a);                                                                               \
    }
RT_PAGED_KERNELS(64)
RT_PAGED_KERNELS(128)
RT_PAGED_KERNELS(256)
