// k_paged_q4.hip — batches over paged caches of 4 bits: the rotary embedding
// with the append of new rows, their way back, and the causal attention.
//
// A group of 32 elements of a head's key or value has one scale word: the step d,
// an f16 of seven significant bits, whose lowest four bits hold the zero point z; a code n in
// 0 .. 15 stands for d·(n − z).  Seven bits times the four of n − z are the eleven
// of an f16: what the codes stand for is one exactly, and the f16 matrix
// cores take it as they take f16 pages.  4.5 bits an element.
//
// A KV head's part of a page of ps positions: ps·HD/2 bytes of codes, then
// ps·HD/32 scale words, so laid out that a lane's operands of the matrix
// cores are one load:
//   keys    codes [ps][HD/8] words of 8 elements, the even ones in the lower half;
//           scales [ps][HD/32];
//   values  per tile of 16 positions: codes [HD/(16·W)][4][16][2][W/4] words, W =
//           4 at head size 64, else 8: word (i, g, c, p, h) has the elements 16·W·i + W·c
//           + 4h .. + 3 of the positions 4g + 2p (lower half) and 4g + 2p + 1; scales
//           [HD/32][16].
// So no byte is two positions', and rows are stored without a look at others.
#include "rt_paged.h"

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// (the type of these pages' elements in rt_paged.h's templates: a byte)
struct Q4 {
    uint8_t b;
};
template <int HD>
struct Q4Layout {
    static constexpr uint32_t W = HD == 64 ? 4 : 8, VN = HD / (16 * W);
    static constexpr uint32_t TILE = RT_PAGED_TILE * HD / 2;    // bytes of a tile's codes
    static constexpr uint32_t SCALES = RT_PAGED_TILE * HD / 16;  // of its scales
    static constexpr uint32_t ROW = HD / 2 + HD / 16;            // of a position
};

// The eight values of a word of codes as four pairs (code k of the lower half, k of the upper).  z: 1024 +
// the zero points, d: the steps of the two halves; z16 = 1024 + 16·z, d16 = d / 16.
// (1024 + n as an f16 has n in its lowest bits, 1024 + 16n four above.)
struct Q4Scale {
    h2_t z, z16, d, d16;
    RT_DEV explicit Q4Scale(uint32_t w) {  // the halves' scale words
        z = __builtin_bit_cast(h2_t, (w & 0x000F000Fu) | 0x64006400u);
        z16 = __builtin_bit_cast(h2_t, (w & 0x000F000Fu) << 4 | 0x64006400u);
        d = __builtin_bit_cast(h2_t, w & 0xFFF0FFF0u);
        d16 = d * (h2_t){(_Float16)0.0625f, (_Float16)0.0625f};
    }
};
RT_DEV void q4_values(uint32_t w, const Q4Scale& s, h2_t (&o)[4]) {
    // (constants known to the compiler would be literals, of which an instruction takes one: two for each of these)
    uint32_t low = 0x000F000Fu, high = 0x00F000F0u, one = 0x64006400u;
    asm("" : "+s"(low), "+s"(high), "+v"(one));
    const uint32_t v = w >> 8;
    o[0] = (__builtin_bit_cast(h2_t, (w & low) | one) - s.z) * s.d;
    o[1] = (__builtin_bit_cast(h2_t, (w & high) | one) - s.z16) * s.d16;
    o[2] = (__builtin_bit_cast(h2_t, (v & low) | one) - s.z) * s.d;
    o[3] = (__builtin_bit_cast(h2_t, (v & high) | one) - s.z16) * s.d16;
}
// The same by way of bytes, for narrow blocks, an instruction or two in thirteen fewer: a byte of 0 .. 15 is
// n·2^-9 as an e4m3 (no exponent, then the first of its exponents: both in steps of 2^-9), and n·d −
// z·d, z·d an f16 exactly, is one fma (the 7B step 34.6 -> 33.8 µs with keys in the order 0, 4, 1, 5, 2, 6, 3, 7,
// which queries take; 34.2 -> 33.6 with values, whose bytes change places first.  Wide blocks are slower for it,
// prompt chunks 59.8 -> 61.2: there a wave waits for its own few words).
struct Q4ByteScale {
    h2_t d, zd;
    RT_DEV explicit Q4ByteScale(uint32_t w) {  // the halves' scale words
        const h2_t one = {(_Float16)1024.0f, (_Float16)1024.0f};
        d = __builtin_bit_cast(h2_t, w & 0xFFF0FFF0u);
        zd = (__builtin_bit_cast(h2_t, (w & 0x000F000Fu) | 0x64006400u) - one) * d;
    }
};
RT_DEV void q4_bytes(uint32_t w, const Q4ByteScale& s, h2_t (&o)[4]) {  // lower four bits, of the bytes 0, 1 and 2, 3; upper
    const uint32_t lo = w & 0x0F0F0F0Fu, hi = w >> 4 & 0x0F0F0F0Fu;
    o[0] = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false));
    o[1] = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true));
    o[2] = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false));
    o[3] = __builtin_bit_cast(h2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true));
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) o[i] = __builtin_elementwise_fma(o[i], s.d, -s.zd);
}
RT_DEV h8_t q4_row_by_fours(uint32_t w, const Q4ByteScale& s) {  // of a key's codes
    h2_t o[4];
    q4_bytes(w, s, o);
    return (h8_t){o[0][0], o[0][1], o[1][0], o[1][1], o[2][0], o[2][1], o[3][0], o[3][1]};
}
RT_DEV void q4_pairs(uint32_t w, const Q4ByteScale& s, h2_t (&o)[4]) {  // as q4_values
    h2_t x[4];
    q4_bytes(__builtin_amdgcn_perm(w, w, 0x03010200u), s, x);
    o[0] = x[0], o[1] = x[2], o[2] = x[1], o[3] = x[3];
}
RT_DEV h8_t q4_row(uint32_t w, const Q4Scale& s) {  // a word of a key's codes, in order
    h2_t o[4];
    q4_values(w, s, o);
    return (h8_t){o[0][0], o[0][1], o[1][0], o[1][1], o[2][0], o[2][1], o[3][0], o[3][1]};
}

template <>
struct PagedView<Q4> {
    const Q4 *k, *v;         // the KV head's part of page 0
    const uint32_t* table;
    uint64_t page_stride;    // bytes
    uint32_t num_pages, ps_shift;
    uint32_t tb, t1;
    uint32_t lo;
    RT_DEV uint32_t page(uint32_t t) const {
        typedef const __attribute__((address_space(4))) uint32_t* sptr_t;  // (a scalar load)
        return t < t1 ? ((sptr_t)table)[(tb + t) * RT_PAGED_TILE >> ps_shift] : num_pages;
    }
    RT_DEV uint32_t slot(uint32_t t) const { return (tb + t) * RT_PAGED_TILE & ((1u << ps_shift) - 1); }
    // byte of a tile's codes; its scales'
    RT_DEV size_t place(uint32_t t, uint32_t page, uint32_t hd) const {
        return page * page_stride + (size_t)slot(t) * (hd / 2);
    }
    RT_DEV size_t scales(size_t off, uint32_t t, uint32_t hd) const {
        return off + ((size_t)(hd / 2) << ps_shift) - (size_t)slot(t) * (hd / 2 - hd / 16);
    }
    template <int HD>
    RT_DEV float value(size_t off, uint32_t t, uint32_t r, uint32_t d) const {
        constexpr uint32_t W = Q4Layout<HD>::W;
        const uint32_t n = (((d / (16 * W) * 4 + r / 4) * 16 + d / W % 16) * 2 + r % 4 / 2) * (W / 4) + d % W / 4;
        const uint32_t s = ((const uint16_t*)(v + scales(off, t, HD)))[d / 32 * 16 + r];
        h2_t o[4];
        q4_values(((const uint32_t*)(v + off))[n], Q4Scale(s | s << 16), o);
        float x = 0.0f;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) x = d % 4 == k ? (float)(r & 1 ? o[k][1] : o[k][0]) : x;
        return x;
    }
    template <int HD>
    static RT_DEV size_t part(uint32_t kvh, uint32_t ps_shift) { return ((size_t)kvh << ps_shift) * Q4Layout<HD>::ROW; }
};

// A tile's operands for the f32 matrix cores (jobs whose sums are not finite), as an f16 page's.
template <int HD>
struct PagedTile<HD, Q4> {
    static constexpr uint32_t KW = 8, KN = HD / 32, VW = Q4Layout<HD>::W, VN = Q4Layout<HD>::VN;
    typedef _Float16 vvec __attribute__((ext_vector_type(VW)));
    h8_t k[KN];
    vvec v[4][VN];
    RT_DEV void load_k(const PagedView<Q4>& w, size_t off, uint32_t t, uint32_t lane) {
        const uint32_t r = lane & 15, g = lane >> 4;
        const uint32_t* c = (const uint32_t*)(w.k + off) + r * (HD / 8) + g;
        const uint16_t* s = (const uint16_t*)(w.k + w.scales(off, t, HD)) + r * (HD / 32);
#pragma unroll
        for (uint32_t i = 0; i < KN; ++i) k[i] = q4_row(c[4 * i], Q4Scale(s[i] * 0x10001u));
    }
    RT_DEV void load_v(const PagedView<Q4>& w, size_t off, uint32_t t, uint32_t lane) {
        const uint32_t c = lane & 15, g = lane >> 4;
        const uint16_t* s = (const uint16_t*)(w.v + w.scales(off, t, HD));
#pragma unroll
        for (uint32_t i = 0; i < VN; ++i)
#pragma unroll
            for (uint32_t p = 0; p < 2; ++p)
#pragma unroll
                for (uint32_t h = 0; h < VW / 4; ++h) {
                    const uint32_t* ss = (const uint32_t*)(s + (16 * VW * i + VW * c) / 32 * 16 + 4 * g + 2 * p);
                    h2_t o[4];
                    q4_values(((const uint32_t*)(w.v + off))[(((i * 4 + g) * 16 + c) * 2 + p) * (VW / 4) + h], Q4Scale(*ss), o);
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) {
                        v[2 * p][i][4 * h + e] = o[e][0];
                        v[2 * p + 1][i][4 * h + e] = o[e][1];
                    }
                }
    }
    RT_DEV void clear(uint32_t pos0, uint32_t lo, uint32_t limx) {
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r)
#pragma unroll
            for (uint32_t i = 0; i < VN; ++i) v[r][i] = pos0 + r < lo || pos0 + r >= limx ? vvec{} : v[r][i];
    }
};

// ───────────────────────────── append, and back ─────────────────────────────
//
// As k_paged_append's: a workgroup a row and group of heads (many rows: all its groups, the
// next one's elements on their way), a thread four elements of a head's
// lower half and the four behind them of its upper.  Eight threads have a group:
// its limits are three steps across lanes.  Bound by the rows' bytes, behind them by the 64 bits:
// 2,068 rows of 28 + 4 + 4 heads of 128 15.7 µs (61 MB, 3.9 TB/s), the way back 4.9.  Few rows: by
// the 64 bits one behind the other (power, sine and cosine, the step's quotient), 4.3 µs where f32 and
// f16 pages take 2.4.
//
// lo = min(0, x), hi = max(0, x); d = (hi − lo) / 15 up to seven bits, 2^-20 at
// least apart; z = −lo/d and n = x/d + z, each to the nearest, n kept within 0 .. 15.
// In 64 bits, keys from their rotation on: in 32 an element in a million goes to the
// code beside its own, and a group in a hundred thousand to another step.
RT_DEV double max8_64(double v) {  // over aligned groups of 8 lanes
    auto from = [&](auto dpp) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        return __builtin_bit_cast(double, (uint64_t)(uint32_t)dpp((int)(b >> 32)) << 32 | (uint32_t)dpp((int)b));
    };
    v = fmax(v, from([](int x) { return dpp_i<DPP_QUAD_PERM(1, 0, 3, 2)>(x); }));
    v = fmax(v, from([](int x) { return dpp_i<DPP_QUAD_PERM(2, 3, 0, 1)>(x); }));
    return fmax(v, from([](int x) { return dpp_i<DPP_ROW_HALF_MIRROR>(x); }));
}
struct Q4Group {
    uint32_t word;    // the scale word
    uint32_t n[4];
};
RT_DEV Q4Group q4_code(const double (&x)[4]) {
    double lo = 0.0, hi = 0.0;
    bool bad = false;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        lo = fmin(lo, x[i]), hi = fmax(hi, x[i]);
        bad |= !(fabs(x[i]) <= 32768.0);
    }
    lo = -max8_64(-lo), hi = max8_64(hi);
    bad = max8(bad ? 1.0f : 0.0f) > 0.0f;
    const double step = (hi - lo) / 15.0;
    // up to six bits behind the leading one; below 2^-14 to multiples of 2^-20
    const double d = step < 6.103515625e-5
                         ? ceil(step * 1048576.0) * 9.5367431640625e-7
                         : __builtin_bit_cast(double, (__builtin_bit_cast(uint64_t, step) + ((1ull << 46) - 1)) & ~((1ull << 46) - 1));
    const double inv = d > 0.0 ? 1.0 / d : 0.0, z = rint(-lo * inv);
    Q4Group g;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) g.n[i] = bad ? 0u : (uint32_t)(float)fmin(fmax(rint(x[i] * inv) + z, 0.0), 15.0);
    g.word = bad ? 0x7E00u : (uint32_t)f2h((float)d) | (uint32_t)(float)z;
    return g;
}
template <int HD>
RT_DEV void q4_store(const PagedBatch& b, uint32_t page, uint32_t kvh, uint32_t slot, bool isv, uint32_t d, const Q4Group& g) {
    constexpr uint32_t W = Q4Layout<HD>::W;
    uint8_t* part = (uint8_t*)(isv ? b.v : b.k) + page * b.page_stride + PagedView<Q4>::part<HD>(kvh, b.ps_shift);
    uint16_t* scales = (uint16_t*)(part + ((size_t)(HD / 2) << b.ps_shift));
    if (isv) {
        const uint32_t r = slot % 16;
        uint16_t* tile = (uint16_t*)(part + (size_t)(slot / 16) * Q4Layout<HD>::TILE);
        const uint32_t n = (((d / (16 * W) * 4 + r / 4) * 16 + d / W % 16) * 2 + r % 4 / 2) * (W / 4) + d % W / 4;
        tile[2 * n + r % 2] = (uint16_t)(g.n[0] | g.n[1] << 4 | g.n[2] << 8 | g.n[3] << 12);
        if (d % 32 == 0) scales[slot / 16 * (HD / 2) + d / 32 * 16 + r] = (uint16_t)g.word;
    } else {
        // (eight elements are two threads')
        const uint32_t mine = g.n[0] | g.n[2] << 4 | g.n[1] << 16 | g.n[3] << 20, next = lane_xor<1>(mine);
        if (d % 8 == 0) ((uint32_t*)part)[(size_t)slot * (HD / 8) + d / 8] = mine | next << 8;
        if (d % 32 == 0) scales[slot * (HD / 32) + d / 32] = (uint16_t)g.word;
    }
}
template <int HD>
RT_DEV void paged_append_q4(const PagedAppendArgs& a) {
    constexpr uint32_t half = HD / 2, TH = half / 4, HW = 256 / TH;  // threads a head, heads a pass
    __shared__ double cs[half], sn[half];
    const PagedBatch& b = a.b;
    const uint32_t row = blockIdx.x, tid = threadIdx.x, ht = tid / TH, d = tid % TH * 4;
    // (a head each group of threads and pass; its elements are on their way while the row's place and angles are
    // found, and heads of values alone need no angles)
    const uint32_t heads = a.H + 2 * b.KVH;
    uint32_t h = blockIdx.y * HW + ht;
    f32x4 lo, hi;
    auto load = [&] {
        if (h >= heads) return;
        const float* src = (h < a.H ? a.q + ((size_t)row * a.H + h) * HD
                            : h < a.H + b.KVH ? a.k + ((size_t)row * b.KVH + h - a.H) * HD
                                              : a.v + ((size_t)row * b.KVH + h - a.H - b.KVH) * HD) + d;
        lo = *(const f32x4*)src, hi = *(const f32x4*)(src + half);
    };
    load();
    const uint32_t s = paged_seq(b, row);
    if (s >= b.n_seqs) return;  // behind the last sequence
    const auto [pos, page] = paged_place(b, s, row);
    if (tid < half && blockIdx.y * HW < a.H + b.KVH) {
        const double turns = (double)pos * exp2(-(double)(2 * tid) / HD * a.log2_theta) * 0.15915494309189535;
        sincospi(2.0 * (turns - rint(turns)), &sn[tid], &cs[tid]);
    }
    lds_barrier();
    const uint32_t slot = pos & ((1u << b.ps_shift) - 1);
    while (h < heads) {
        const uint32_t me = h;
        const f32x4 l = lo, u = hi;
        h += gridDim.y * HW;
        load();
        if (me < a.H) {
            f32x4 c4, s4;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) c4[i] = (float)cs[d + i], s4[i] = (float)sn[d + i];
            float* o = a.q_out + ((size_t)row * a.H + me) * HD + d;
            *(f32x4*)o = l * c4 - u * s4;
            *(f32x4*)(o + half) = l * s4 + u * c4;
        } else if (page < b.num_pages) {
            const bool isv = me >= a.H + b.KVH;
            const uint32_t kh = me - a.H - (isv ? b.KVH : 0);
            double x[4], y[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                x[i] = (double)l[i], y[i] = (double)u[i];
                if (!isv) {
                    const double c = cs[d + i], w = sn[d + i], z = x[i];
                    x[i] = z * c - y[i] * w;
                    y[i] = z * w + y[i] * c;
                }
            }
            q4_store<HD>(b, page, kh, slot, isv, d, q4_code(x));
            q4_store<HD>(b, page, kh, slot, isv, d + half, q4_code(y));
        }
    }
}

// Four elements of a row's key or value, from d on.
template <int HD>
RT_DEV f32x4 q4_load(const PagedBatch& b, uint32_t page, uint32_t kvh, uint32_t slot, bool isv, uint32_t d) {
    constexpr uint32_t W = Q4Layout<HD>::W;
    const uint8_t* part = (const uint8_t*)(isv ? b.v : b.k) + page * b.page_stride + PagedView<Q4>::part<HD>(kvh, b.ps_shift);
    const uint16_t* scales = (const uint16_t*)(part + ((size_t)(HD / 2) << b.ps_shift));
    f32x4 x;
    h2_t o[4];
    if (isv) {
        const uint32_t r = slot % 16;
        const uint32_t n = (((d / (16 * W) * 4 + r / 4) * 16 + d / W % 16) * 2 + r % 4 / 2) * (W / 4) + d % W / 4;
        const uint32_t w = ((const uint16_t*)(part + (size_t)(slot / 16) * Q4Layout<HD>::TILE))[2 * n + r % 2];
        q4_values(w, Q4Scale(scales[slot / 16 * (HD / 2) + d / 32 * 16 + r]), o);
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) x[i] = (float)o[i][0];
    } else {
        const uint32_t w = ((const uint32_t*)part)[(size_t)slot * (HD / 8) + d / 8] >> (d % 8 ? 8 : 0);
        q4_values(w, Q4Scale(scales[slot * (HD / 32) + d / 32] * 0x10001u), o);
        x = (f32x4){(float)o[0][0], (float)o[0][1], (float)o[1][0], (float)o[1][1]};
    }
    return x;
}
template <class O>
RT_DEV void paged_gather_q4(const PagedGatherArgs& a) {
    paged_gather<O>(a, [&](uint32_t page, uint32_t kvh, uint32_t slot, bool isv, uint32_t d) {
        return a.head_dim == 64    ? q4_load<64>(a.b, page, kvh, slot, isv, d)
               : a.head_dim == 128 ? q4_load<128>(a.b, page, kvh, slot, isv, d)
                                   : q4_load<256>(a.b, page, kvh, slot, isv, d);
    });
}

// ───────────────────────────── attention ─────────────────────────────
//
// As over f16 pages: Sᵀ = K·Qᵀ, Oᵀ = Vᵀ·Pᵀ with a running maximum and sum, q and the
// weights as pairs of f16.  A code's f16 is exact, so that its step and zero point
// need no sums of their own; but each code is made f16 once in every block that reads it,
// which bounds narrow blocks beside memory: 32 sequences of up to 16,000 positions of 4 KV heads of
// 128 with 7 query heads each 33 µs for 108 MB (3.3 TB/s), their loads and launches alone 26–28.
// Of narrow blocks the parts meet in a launch of their own (paged_meet) where there may be many.

// A wave's own ring of stages in LDS, a turn's two tiles each: codes of keys and values as their
// lanes' operands, scale words as they are.  A lane reads what it, or its wave, brought: no
// barriers; and any number of turns may be on their way, waited for by their number of loads (loads
// into registers, two turns ahead, are waited for one too early at the loop's end).
template <int HD>
struct Q4Stage {
    static constexpr uint32_t W = Q4Layout<HD>::W, VN = Q4Layout<HD>::VN, KN = HD / 32;
    static constexpr uint32_t CW = HD == 64 ? 2 : 4;      // words of a read of codes
    static constexpr uint32_t CODES = HD * 8, SCALES = HD;  // bytes of a tile's keys, values
    static constexpr uint32_t LEN = 4 * (CODES + SCALES), N = HD == 256 ? 3 : 4;
    static constexpr uint32_t LOADS = HD == 64 ? 3 : HD == 128 ? 6 : 12;
};
template <int HD>
struct PagedWave<HD, Q4> {
    static constexpr uint32_t LDS = Q4Stage<HD>::N * Q4Stage<HD>::LEN / 4;
    static constexpr bool HALF = true, MAY_NOTE = true;
    static_assert(LDS >= 16 * (HD + 4), "the outputs fit");
};
// 16 or 4 bytes a lane to LDS, lane 0's at byte `at`, each next behind it: from p (the lane's own), and
// from off (the lane's own) behind p.
template <uint32_t BYTES>
RT_DEV void q4_bring(const void* p, uint32_t at) {
    if constexpr (BYTES == 16)
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(p), "s"(at) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(at) : "memory", "m0");
}
RT_DEV void q4_bring16(const void* p, uint32_t off, uint32_t at) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(p), "s"(at) : "memory", "m0");
}
RT_DEV void q4_bring4(const void* p, uint32_t off, uint32_t at) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(p), "s"(at) : "memory", "m0");
}
// waits until at most n of the wave's last `most` stages are on their way
template <uint32_t LOADS, uint32_t MOST>
RT_DEV void q4_stages_left(uint32_t n) {
    constexpr auto wait = [](uint32_t c) constexpr { return (c & 15) | (c >> 4) << 14 | 7 << 4 | 15 << 8; };
    if constexpr (MOST > 0) {
        if (n >= MOST) __builtin_amdgcn_s_waitcnt(wait(MOST * LOADS));
        else q4_stages_left<LOADS, MOST - 1>(n);
    } else {
        __builtin_amdgcn_s_waitcnt(wait(0));
    }
}

// A turn's operands, as a lane reads them from its stage: keys, of position l % 16 the elements
// HD/4·(l / 16) ..; values, of positions 4·(l / 16) .. + 3, W of every 16·W elements from W·(l % 16) on.
template <int HD>
struct Q4Raw {
    typedef Q4Stage<HD> S;
    static constexpr uint32_t W = S::W, VN = S::VN, KN = S::KN, CW = S::CW;
    typedef uint32_t cvec __attribute__((ext_vector_type(CW)));
    cvec k[KN / CW], v[KN / CW];
    uint32_t ks;        // at head size 256 two words
    u32x2 vs[VN];
    RT_DEV void keys(const uint8_t* p, const uint8_t* s, uint32_t lane) {
        const uint32_t c = lane & 15, g = lane >> 4;
        p += HD == 64 ? c * 32 + g * 8 : lane * 16;
#pragma unroll
        for (uint32_t i = 0; i < KN / CW; ++i) k[i] = *(const cvec*)(p + i * 1024);
        s += c * (HD / 16) + (HD == 256 ? 4 * g : HD == 128 ? 2 * g : g / 2 * 2);
        if constexpr (HD == 256) ks = *(const uint32_t*)s;
        else ks = *(const uint16_t*)s;
    }
    RT_DEV void values(const uint8_t* p, const uint8_t* s, uint32_t lane) {
        const uint32_t c = lane & 15, g = lane >> 4;
        p += lane * CW * 4;
        s += W * c / 32 * 32 + 8 * g;
#pragma unroll
        for (uint32_t i = 0; i < KN / CW; ++i) v[i] = *(const cvec*)(p + i * 1024);
#pragma unroll
        for (uint32_t i = 0; i < VN; ++i) vs[i] = *(const u32x2*)(s + i * 16 * W);
    }
    // positions that no column sees may hold anything: steps of zero (a code is always finite)
    RT_DEV void clear(uint32_t pos0, uint32_t lo, uint32_t limx) {
#pragma unroll
        for (uint32_t r = 0; r < 4; ++r)
            if (pos0 + r < lo || pos0 + r >= limx)
#pragma unroll
                for (uint32_t i = 0; i < VN; ++i) vs[i][r / 2] &= r % 2 ? 0x0000FFFFu : 0xFFFF0000u;
    }
    RT_DEV uint32_t kscale(uint32_t i) const {  // of the key's words i, twice
        if constexpr (HD == 256) return i < KN / 2 ? (ks & 0xFFFFu) | ks << 16 : ks >> 16 | (ks & 0xFFFF0000u);
        return ks | ks << 16;
    }
};

// The tiles t0, t0 + 1, t0 + step, ... for 16 columns, as f16 pages': queries and
// weights as pairs of f16, two tiles a turn.  A tile without a page is read from the
// pool's first and seen by none.  HALF: eight columns, the upper parts of queries and weights in
// the lanes of columns 0 .. 7, the lower ones in those of 8 .. 15: one product instead of two.
template <int HD, bool HALF>
RT_DEV void q4_chunk(PagedAcc<HD, Q4>& acc, const PagedView<Q4>& v, const float* q, float scale2, uint32_t t0,
                     uint32_t step, uint32_t lim, uint32_t limn, uint32_t limx, float* lds) {
    constexpr int ROW_ROR8 = 0x128;  // the lane of the column eight away
    typedef Q4Stage<HD> S;
    typedef Q4Raw<HD> Raw;
    constexpr uint32_t KN = S::KN, VW = S::W, VN = S::VN, CW = S::CW, N = S::N;
    const uint32_t lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const uint32_t turns = t0 < v.t1 ? (v.t1 - t0 + step - 1) / step : 0;
    // the pages of 64 turns' tiles, a turn a lane
    uint32_t ids[2];
    auto ids_from = [&](uint32_t i0) {
        const uint32_t t = t0 + (i0 + lane) * step;
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u)
            ids[u] = i0 + lane < turns && t + u < v.t1 ? v.table[(v.tb + t + u) * RT_PAGED_TILE >> v.ps_shift] : v.num_pages;
    };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const float*)lds);
    // what a lane brings, from a tile's codes (scale words) on
    const uint8_t *kc, *sc;
    const uint32_t ko = HD == 128 ? c * 64 + g * 16 : c * 128 + g * 32, vo = lane * 16;
    if constexpr (HD == 64) {  // keys by the lower half of the lanes; both tiles' scales at once
        kc = (const uint8_t*)(lane < 32 ? v.k : v.v) + lane % 32 * 16;
        sc = (const uint8_t*)(lane & 16 ? v.v : v.k) + c * 4;
    } else {
        sc = (const uint8_t*)(HD == 128 && lane >= 32 ? v.v : v.k) + (HD == 128 ? lane % 32 * 4 : lane * 4);
    }
    const size_t s0 = (size_t)(HD / 2) << v.ps_shift;  // of a page's scale words
    // turn i's tiles into stage i % N; whether they have a page, a bit each
    auto bring = [&](uint32_t i) {
        const uint32_t t = t0 + i * step, st = lds0 + i % N * S::LEN;
        size_t off[2], so[2];
        uint32_t there = 0;
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
            const uint32_t page = __builtin_amdgcn_readlane(ids[u], i & 63);
            there |= page < v.num_pages ? 1u << u : 0u;
            const size_t at = (page < v.num_pages ? page : 0) * v.page_stride;
            off[u] = at + (size_t)v.slot(t + u) * (HD / 2);
            so[u] = at + s0 + (size_t)v.slot(t + u) * (HD / 16);
            asm("" : "+s"(off[u]), "+s"(so[u]));  // (sums of all lanes', not of each)
        }
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) {
            const uint32_t to = st + u * 2 * S::CODES;
            if constexpr (HD == 64) {
                q4_bring<16>(kc + off[u], to);
            } else {
#pragma unroll
                for (uint32_t x = 0; x < HD / 128; ++x) {
                    q4_bring16((const uint8_t*)v.k + off[u], ko + x * 16, to + x * 1024);
                    q4_bring16((const uint8_t*)v.v + off[u], vo + x * 1024, to + S::CODES + x * 1024);
                }
            }
        }
        const uint32_t to = st + 4 * S::CODES;
        if constexpr (HD == 64) {
            q4_bring<4>(sc + (lane < 32 ? so[0] : so[1]), to);
        } else {
#pragma unroll
            for (uint32_t u = 0; u < 2; ++u) {
                q4_bring<4>(sc + so[u], to + u * 2 * S::SCALES);
                if constexpr (HD == 256) q4_bring<4>((const uint8_t*)v.v + lane * 4 + so[u], to + (u * 2 + 1) * S::SCALES);
            }
        }
        return there;
    };
    uint32_t here = 0;  // bring()'s bits of turns i .. i + N - 1
    if (turns) {
        ids_from(0);
#pragma unroll
        for (uint32_t i = 0; i < N - 1; ++i)
            if (i < turns) here |= bring(i) << 2 * i;
    }
    h8_t qh[KN], ql[KN];
    const float qs = paged_query<HD, true>(q, scale2, qh, ql);
#pragma unroll
    for (uint32_t n = 0; n < KN; ++n) {  // (as the keys come)
        qh[n] = __builtin_shufflevector(qh[n], qh[n], 0, 4, 1, 5, 2, 6, 3, 7);
        ql[n] = __builtin_shufflevector(ql[n], ql[n], 0, 4, 1, 5, 2, 6, 3, 7);
    }
    if constexpr (HALF)
#pragma unroll
        for (uint32_t n = 0; n < KN; ++n) qh[n] = c < 8 ? qh[n] : ql[n];
    acc.start();
    // turn i's operands out of its stage, on their way while the turn before is computed; the N − 2 stages behind it
    // may still be on theirs
    auto take = [&](uint32_t i, Raw (&raw)[2]) {
        q4_stages_left<S::LOADS, N - 2>(turns - 1 - i);
        asm volatile("" ::: "memory");
        const uint8_t* st = (const uint8_t*)lds + i % N * S::LEN;
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u) raw[u].keys(st + u * 2 * S::CODES, st + 4 * S::CODES + u * 2 * S::SCALES, lane);
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u)
            raw[u].values(st + (u * 2 + 1) * S::CODES, st + 4 * S::CODES + (u * 2 + 1) * S::SCALES, lane);
    };
    auto turn = [&](uint32_t i, Raw (&raw)[2], Raw (&next)[2]) {
        const uint32_t p0 = (v.tb + t0 + i * step) * RT_PAGED_TILE;
        const bool there[2] = {(here & 1) != 0, (here & 2) != 0};
        here >>= 2;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4 | 0 << 8);  // (LDS: this turn's stage is read)
        if (i + N - 1 < turns) {  // (into the stage before this one)
            if ((i + N - 1) % 64 == 0) ids_from(i + N - 1);
            here |= bring(i + N - 1) << 2 * (N - 2);
        }
        if (i + 1 < turns) take(i + 1, next);  // (N − 2 stages are brought behind it, or all there are)
        const bool edge = p0 < v.lo || p0 + 2 * RT_PAGED_TILE > limn || !there[0] || !there[1];
        f32x4 sa[2] = {}, sb[2] = {};
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u)
#pragma unroll
            for (uint32_t n = 0; n < KN; ++n) {
                const h8_t k = q4_row_by_fours(raw[u].k[n / CW][n % CW], Q4ByteScale(raw[u].kscale(n)));
                sa[u] = mfma32(k, qh[n], sa[u]);
                if constexpr (!HALF) sb[u] = mfma32(k, ql[n], sb[u]);
            }
        // HALF: the scores of the first tile in the lanes of columns 0 .. 7, of the second in the others'
        constexpr uint32_t P = HALF ? 4 : 8;
        float p[P];
        if constexpr (HALF) {
#pragma unroll
            for (uint32_t r = 0; r < 4; ++r) p[r] = (c < 8 ? sa[0][r] : sa[1][r]) + dpp_f<ROW_ROR8>(c < 8 ? sa[1][r] : sa[0][r]);
        } else {
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) p[r] = sa[r / 4][r % 4] + sb[r / 4][r % 4];
        }
        if (edge) {
#pragma unroll
            for (uint32_t r = 0; r < P; ++r) {
                const uint32_t u = HALF ? c / 8 : r / 4, pos = p0 + 16 * u + 4 * g + r % 4;
                if (pos < v.lo || pos >= lim || !(u ? there[1] : there[0])) p[r] = -__builtin_huge_valf();
            }
#pragma unroll
            for (uint32_t u = 0; u < 2; ++u) raw[u].clear(p0 + 16 * u + 4 * g, v.lo, there[u] ? limx : 0);
        }
        acc.template weigh<P, HALF>(p, qs);
        h8_t ph, pl;
        if constexpr (HALF) {
            // the upper parts of all eight to the lanes of columns 0 .. 7, the lower ones to the others
            h4_t hi, lo;
            split_weights_of<4>(p, hi, lo);
            const u32x2 h2 = __builtin_bit_cast(u32x2, hi), l2 = __builtin_bit_cast(u32x2, lo);
            u32x4 w;
#pragma unroll
            for (uint32_t x = 0; x < 2; ++x) {
                const uint32_t own = c < 8 ? h2[x] : l2[x], other = (uint32_t)dpp_i<ROW_ROR8>((int)(c < 8 ? l2[x] : h2[x]));
                w[x] = c < 8 ? own : other;
                w[2 + x] = c < 8 ? other : own;
            }
            ph = __builtin_bit_cast(h8_t, w);
        } else {
            split_weights(p, ph, pl);
        }
#pragma unroll
        for (uint32_t n = 0; n < VN; ++n)
#pragma unroll
            for (uint32_t h = 0; h < VW / 4; ++h) {
                h2_t o[4][4];  // of the pairs of positions, the elements 4h ..
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) {
                    const uint32_t m = (n * 2 + x % 2) * (VW / 4) + h;
                    q4_pairs(raw[x / 2].v[m / CW][m % CW], Q4ByteScale(raw[x / 2].vs[n][x % 2]), o[x]);
                }
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const h8_t a = {o[0][e][0], o[0][e][1], o[1][e][0], o[1][e][1],
                                    o[2][e][0], o[2][e][1], o[3][e][0], o[3][e][1]};
                    acc.o[n][4 * h + e] = mfma32(a, ph, acc.o[n][4 * h + e]);
                    if constexpr (!HALF) acc.o[n][4 * h + e] = mfma32(a, pl, acc.o[n][4 * h + e]);
                }
            }
    };
    Raw even[2], odd[2];
    if (turns) take(0, even);
    for (uint32_t i = 0; i < turns; i += 2) {
        turn(i, even, odd);
        if (i + 1 < turns) turn(i + 1, odd, even);
    }
    if constexpr (HALF)
#pragma unroll
        for (uint32_t n = 0; n < VN; ++n)
#pragma unroll
            for (uint32_t e = 0; e < VW; ++e)
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x) acc.o[n][e][x] += dpp_f<ROW_ROR8>(acc.o[n][e][x]);
    if constexpr (HALF) acc.l += dpp_f<ROW_ROR8>(acc.l);
    acc.join();
}
template <int HD>
RT_DEV void paged_pairs(PagedAcc<HD, Q4>& acc, const PagedView<Q4>& v, const float* q, float scale2, uint32_t t0,
                      uint32_t step, uint32_t lim, uint32_t limn, uint32_t limx, float* lds, bool half) {
    if (half) q4_chunk<HD, true>(acc, v, q, scale2, t0, step, lim, limn, limx, lds);
    else q4_chunk<HD, false>(acc, v, q, scale2, t0, step, lim, limn, limx, lds);
}

// Wide blocks: the codes become f16 on their way to LDS, once for the block's 128 columns; from
// there on they are f16 pages.  Two waves have the keys of a turn's two tiles, two the values, each
// from a ring of its own that is brought three turns ahead (one turn ahead into registers, the turns waited for
// memory: prompt chunks 62 µs for 61); a stage is written while the one before is computed.
template <int HD>
struct PagedFeed<HD, Q4> {
    typedef PagedStage<HD> Stage;
    typedef Q4Raw<HD> Raw;
    static constexpr uint32_t N = 2, W = Q4Layout<HD>::W, VN = Q4Layout<HD>::VN, KN = HD / 32, CW = Raw::CW;
    static constexpr uint32_t CODES = HD * 8, SCALES = HD, RING = 4;  // bytes of a tile's; turns
    static constexpr uint32_t LOADS = HD == 256 ? 3 : 2;
    static_assert(N * Stage::LEN * 16 + RT_PAGED_WAVES * RING * (CODES + SCALES) <= Stage::N * Stage::LEN * 16, "LDS");
    const PagedView<Q4>& v;
    h8_t* lds;
    uint32_t t0, step, turns, limx, here = 0;  // here: bring()'s bits of turns i .. i + 4
    uint32_t ring;     // the wave's, in LDS
    const uint8_t* mine;  // its keys, or values
    uint32_t ids[2];   // the pages of 64 turns' tiles, a turn a lane
    RT_DEV PagedFeed(const PagedView<Q4>& v, h8_t* lds, uint32_t t0, uint32_t step, uint32_t turns, uint32_t limx)
        : v(v), lds(lds), t0(t0), step(step), turns(turns), limx(limx) {
        ring = N * Stage::LEN * 16 + wave() * RING * (CODES + SCALES);
        mine = (const uint8_t*)(wave() < 2 ? v.k : v.v);
    }
    RT_DEV uint32_t wave() const { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
    RT_DEV void ids_from(uint32_t i0) {
        const uint32_t lane = threadIdx.x & 63, t = t0 + (i0 + lane) * step;
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u)
            ids[u] = i0 + lane < turns && t + u < v.t1 ? v.table[(v.tb + t + u) * RT_PAGED_TILE >> v.ps_shift] : v.num_pages;
    }
    // the wave's part of turn i into its ring; whether the turn's tiles have a page
    RT_DEV uint32_t bring(uint32_t i) {
        const uint32_t lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, u = wave() & 1, t = t0 + i * step + u;
        const uint32_t id0 = __builtin_amdgcn_readlane(ids[0], i & 63), id1 = __builtin_amdgcn_readlane(ids[1], i & 63);
        const uint32_t page = u ? id1 : id0;
        const size_t at = (page < v.num_pages ? page : 0) * v.page_stride;
        const uint8_t* codes = mine + at + (size_t)v.slot(t) * (HD / 2);
        const uint8_t* scales = mine + at + ((size_t)(HD / 2) << v.ps_shift) + (size_t)v.slot(t) * (HD / 16);
        const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) const h8_t*)lds);
        const uint32_t to = lds0 + ring + i % RING * (CODES + SCALES);
        // (of 128 and 256 the keys as their lanes' operands; of 64 both as they are, 32 lanes' worth)
        const uint32_t off = wave() >= 2 || HD == 64 ? lane * 16 : HD == 128 ? c * 64 + g * 16 : c * 128 + g * 32;
        if constexpr (HD == 64) {
            if (lane < 32) q4_bring16(codes, off, to);
        } else {
#pragma unroll
            for (uint32_t x = 0; x < HD / 128; ++x) q4_bring16(codes, off + x * (wave() < 2 ? 16 : 1024), to + x * 1024);
        }
        if (lane < HD / 4) q4_bring4(scales, lane * 4, to + CODES);
        return (id0 < v.num_pages ? 1u : 0u) | (id1 < v.num_pages ? 2u : 0u);
    }
    // and from there as f16 into stage i % N; positions that no column sees may hold anything: steps of zero
    RT_DEV void put(uint32_t i, uint32_t there) {
        const uint32_t lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, u = wave() & 1;
        const uint8_t* from = (const uint8_t*)lds + ring + i % RING * (CODES + SCALES);
        h8_t* st = lds + i % N * Stage::LEN;
        q4_stages_left<LOADS, RING - 1>(turns - 1 - i);
        asm volatile("" ::: "memory");
        Raw raw;
        if (wave() < 2) {
            raw.keys(from, from + CODES, lane);
#pragma unroll
            for (uint32_t n = 0; n < KN; ++n)
                st[Stage::piece(16 * u + c, KN * g + n)] = q4_row(raw.k[n / CW][n % CW], Q4Scale(raw.kscale(n)));
            return;
        }
        raw.values(from, from + CODES, lane);
        const uint32_t p0 = (v.tb + t0 + i * step + u) * RT_PAGED_TILE;
        if (p0 < v.lo || p0 + RT_PAGED_TILE > limx || !(there >> u & 1)) raw.clear(p0 + 4 * g, v.lo, there >> u & 1 ? limx : 0);
#pragma unroll
        for (uint32_t n = 0; n < VN; ++n)
#pragma unroll
            for (uint32_t p = 0; p < 2; ++p) {  // two positions
                h2_t o[W / 4][4];
                const Q4Scale s(raw.vs[n][p]);
#pragma unroll
                for (uint32_t h = 0; h < W / 4; ++h) {
                    const uint32_t m = (n * 2 + p) * (W / 4) + h;
                    q4_values(raw.v[m / CW][m % CW], s, o[h]);
                }
#pragma unroll
                for (uint32_t x = 0; x < 2; ++x) {
                    const uint32_t row = 32 + 16 * u + 4 * g + 2 * p + x;
                    if constexpr (W == 8) {
                        st[Stage::piece(row, 16 * n + c)] =
                            (h8_t){o[0][0][x], o[0][1][x], o[0][2][x], o[0][3][x], o[1][0][x], o[1][1][x], o[1][2][x], o[1][3][x]};
                    } else {
                        ((h4_t*)(st + Stage::piece(row, c / 2)))[c & 1] = (h4_t){o[0][0][x], o[0][1][x], o[0][2][x], o[0][3][x]};
                    }
                }
            }
    }
    RT_DEV void start() {
        if (!turns) return;
#pragma unroll
        for (uint32_t i = 0; i < RING; ++i)
            if (i < turns) here |= bring(i) << 2 * i;
        put(0, here & 3);
    }
    RT_DEV uint32_t turn(uint32_t i) {
        const uint32_t there = here & 3;
        here >>= 2;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4 | 0 << 8);  // (LDS: its part of this stage is written, of the ring read)
        __builtin_amdgcn_s_barrier();  // (this stage is there, the one before is read)
        asm volatile("" ::: "memory");
        if (i + RING < turns) {
            if ((i + RING) % 64 == 0) ids_from(i + RING);
            here |= bring(i + RING) << 2 * (RING - 1);
        }
        if (i + 1 < turns) put(i + 1, here & 3);
        return there;
    }
};

// As paged_merge, of many chunks: a workgroup a (row, head), HD / 4 threads a group, each group every
// G-th chunk, as many at a time as there are; the groups meet in LDS.  (Four at a time for any number: the 7B step
// 33.7 µs for 33.3, 200,005 positions 37.8 for 37.1.  40 rows over a prefix of 8,192 positions in 30 chunks: 7.2 µs as
// paged_merge, with a thread's chunks one batch after another.)
template <int HD, bool WIDE>
RT_DEV void paged_meet(const PagedAttnArgs& a) {
    constexpr uint32_t TH = HD / 4, G = 256 / TH, SR = paged_slot_rows<WIDE>();
    __shared__ f32x4 os[G][TH];
    __shared__ float ms[G], ls[G];
    const PagedBatch& b = a.b;
    const uint32_t rh = blockIdx.x, grp = threadIdx.x / TH, t = threadIdx.x % TH;
    const uint32_t rows = b.row_start ? min(b.row_start[b.n_seqs], b.rows) : min(b.n_seqs, b.rows);
    if (rh >= rows * a.H) return;
    const uint32_t kvh = rh % a.H / (a.H / b.KVH);
    const u32x4 in = *(const u32x4*)(a.info + (size_t)rh * 4);
    const uint32_t n0 = in[1] / SR, n = n0 + (a.shared_len ? in[3] / SR : 0);
    if (!a.shared_len && n0 == 1) return;  // (written whole)
    if (in[0] >= a.jobs || n0 > a.jobs - in[0] || (n > n0 && (in[2] >= a.jobs || n - n0 > a.jobs - in[2]))) return;
    const float NEG = -__builtin_huge_valf();
    float M = NEG, L = 0.0f;
    f32x4 o = {0, 0, 0, 0};
    auto take = [&]<uint32_t BATCH>(uint32_t x0) {  // chunks x0, x0 + G, ..: their loads at once
        float mc[BATCH], lc[BATCH], mx = M;
        f32x4 oc[BATCH];
#pragma unroll
        for (uint32_t u = 0; u < BATCH; ++u) {
            const uint32_t x = min(x0 + u * G, n - 1), job = x < n0 ? in[0] + x : in[2] + x - n0;
            const size_t slot = ((size_t)job * b.KVH + kvh) * SR + (x < n0 ? in[1] : in[3]) % SR;
            mc[u] = a.ml[2 * slot], lc[u] = a.ml[2 * slot + 1];
            oc[u] = *(const f32x4*)(a.part + slot * HD + 4 * t);
        }
#pragma unroll
        for (uint32_t u = 0; u < BATCH; ++u) mx = fmaxf(mx, mc[u]);
        const float md = mx == NEG ? 0.0f : mx, f0 = __builtin_amdgcn_exp2f(M - md);
        M = mx;
        L *= f0;
        o *= f0;
#pragma unroll
        for (uint32_t u = 0; u < BATCH; ++u) {
            if (x0 + u * G >= n) continue;
            const float f = __builtin_amdgcn_exp2f(mc[u] - md);
            L = fmaf(f, lc[u], L);
            o += f * oc[u];
        }
    };
    uint32_t x0 = grp;
    for (; x0 + 7 * G < n; x0 += 8 * G) take.template operator()<8>(x0);
    for (; x0 + 2 * G < n; x0 += 4 * G) take.template operator()<4>(x0);
    for (; x0 < n; x0 += 2 * G) take.template operator()<2>(x0);
    os[grp][t] = o;
    if (t == 0) ms[grp] = M, ls[grp] = L;
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (uint32_t g = 1; g < G; ++g) M = fmaxf(M, ms[g]);
    const float md = M == NEG ? 0.0f : M;
    L = 0.0f;
    o = f32x4{0, 0, 0, 0};
#pragma unroll
    for (uint32_t g = 0; g < G; ++g) {
        const float f = __builtin_amdgcn_exp2f(ms[g] - md);
        L = fmaf(f, ls[g], L);
        o += f * os[g][t];
    }
    *(f32x4*)(a.out + (size_t)rh * HD + 4 * t) = L == 0.0f ? f32x4{0, 0, 0, 0} : o / L;
}

#define RT_PAGED_Q4_KERNELS(HD)                                                                           \
    extern "C" __global__ void __launch_bounds__(256) k_paged_append_q4_hd##HD(PagedAppendArgs a) {      \
        paged_append_q4<HD>(a);                                                                           \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) k_paged_attn_q4_hd##HD(PagedAttnArgs a) { \
        paged_attn<HD, Q4, false>(a);                                                                     \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256, HD == 256 ? 1 : 2) k_paged_attn_q4w_hd##HD(PagedAttnArgs a) { \
        paged_attn<HD, Q4, true>(a);                                                                      \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) k_paged_meet_hd##HD(PagedAttnArgs a) {             \
        paged_meet<HD, false>(a);                                                                         \
    }                                                                                                     \
    extern "C" __global__ void __launch_bounds__(256) k_paged_meetw_hd##HD(PagedAttnArgs a) {            \
        paged_meet<HD, true>(a);                                                                          \
    }
RT_PAGED_Q4_KERNELS(64)
RT_PAGED_Q4_KERNELS(128)
RT_PAGED_Q4_KERNELS(256)
extern "C" __global__ void __launch_bounds__(256) k_paged_gather_q4_f32(PagedGatherArgs a) { paged_gather_q4<float>(a); }
extern "C" __global__ void __launch_bounds__(256) k_paged_gather_q4_f16(PagedGatherArgs a) { paged_gather_q4<_Float16>(a); }
