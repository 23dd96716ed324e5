// Serving attention around the decode projections, for gfx950: the q|k|v projection's k and v
// rotated and appended to a paged cache, and attention over that cache (sliding window, sink
// tokens, a prefix shared by the whole batch).
//
// A sequence's position j lies in page table[b][j / page_size], slot j % page_size.  The query
// token i of the n that a call brings for sequence b is at position p = lens[b] - n + i (lens
// counts the call's own tokens) and sees key j <= p where j > p - window or j < sinks.
// Table, lengths and query offsets are device data, so every kernel bounds them itself: a table
// entry that names no page of the cache stands for keys that are not there.

#include "nf4_common.h"

namespace {

struct Cache {
    uint16_t *k, *v;
    int64_t page_stride, slot_stride, head_stride;
    const int32_t *table;
    int64_t ld_table;
    const int32_t *lens;
    const int32_t *cu;  // query offsets [batch + 1], or null: tokens / batch each
    int pages, page_shift, cap, batch, n_kv, tokens, uniform;
};

// Query tokens [q0, q0 + n) of sequence b and the position of the first.  Sequence `batch`
// stands for the tokens past the last offset: positions below zero, which see nothing.
struct Seq {
    int q0, n, p0;
};

__device__ __forceinline__ int clamp_tok(const Cache &c, int v) {
    return v < 0 ? 0 : (v > c.tokens ? c.tokens : v);
}

__device__ __forceinline__ Seq seq_at(const Cache &c, int b) {
    Seq s;
    if (c.cu) {
        s.q0 = b == 0 ? 0 : clamp_tok(c, c.cu[b]);
        s.n = (b == c.batch ? c.tokens : clamp_tok(c, c.cu[b + 1])) - s.q0;
        s.n = s.n < 0 ? 0 : s.n;
    } else {
        s.q0 = b * c.uniform;
        s.n = b == c.batch ? 0 : c.uniform;
    }
    const int len = b == c.batch ? 0 : c.lens[b];
    s.p0 = len < 0 ? -s.n : len - s.n;
    return s;
}

// The same for a b that is the wave's, in scalar registers (loop bounds and branches then are
// scalar ones).
__device__ __forceinline__ Seq seq_uniform(const Cache &c, int b) {
    Seq s = seq_at(c, b);
    s.q0 = __builtin_amdgcn_readfirstlane(s.q0);
    s.n = __builtin_amdgcn_readfirstlane(s.n);
    s.p0 = __builtin_amdgcn_readfirstlane(s.p0);
    return s;
}

// The sequence of token t: with offsets, how many sequences end at or before it (64 at a time).
__device__ __forceinline__ int seq_of_token(const Cache &c, int t) {
    if (!c.cu) return t / c.uniform;
    int b = 0;
    for (int i = 0; i < c.batch; i += 64) {
        const int j = i + (threadIdx.x & 63);
        const bool past = j < c.batch && c.cu[j + 1] <= t;
        const uint64_t m = __ballot(past);
        b += __popcll(m);
        if (~m) break;
    }
    return __builtin_amdgcn_readfirstlane(b);
}

// Offset of position pos of sequence b, key/value head 0, or -1 where the table names no page.
__device__ __forceinline__ int64_t slot_of(const Cache &c, int b, int pos) {
    const int page = c.table[b * c.ld_table + (pos >> c.page_shift)];
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(c.pages)) return -1;
    return page * c.page_stride + (pos & ((1 << c.page_shift) - 1)) * c.slot_stride;
}

template <int DT>
__device__ __forceinline__ float f32_of(uint32_t bits) {
    if constexpr (DT == NF4_BF16) return __uint_as_float(bits << 16);
    else return static_cast<float>(__builtin_bit_cast(half_t, static_cast<uint16_t>(bits)));
}

template <int DT>
__device__ __forceinline__ void unpack8(const u32x4_t &r, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = f32_of<DT>(r[i] & 0xffffu);
        v[2 * i + 1] = f32_of<DT>(r[i] >> 16);
    }
}

template <int DT>
__device__ __forceinline__ u32x4_t pack8(const float (&v)[8]) {
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = round16<DT>(v[2 * i]) | (static_cast<uint32_t>(round16<DT>(v[2 * i + 1])) << 16);
    return r;
}

// ------------------------------------------------------------------------------- append

constexpr int kAppendThreads = 256;

// One workgroup per token.  A thread takes 8 rotary pairs of a head (16 bytes of its low half
// and 16 of its high half): lo' = lo cos - hi sin, hi' = hi cos + lo sin in fp32, each rounded
// once; v heads are copied the same way.  Bound by memory: 8081 tokens of 28 + 4 + 4 heads, 153 MB,
// in 28.2 us (5.4 TB/s); a step of one token is its launch, 2.5 us.
template <int DT>
__global__ __launch_bounds__(kAppendThreads) void paged_append_kernel(
    const Cache c, const uint16_t *qkv, int64_t ld, const float *cs, const float *sn, int rope_rows,
    uint16_t *qo, int n_heads, int head_dim) {
    const int t = blockIdx.x;
    const int b = seq_of_token(c, t), half = head_dim / 2, per = head_dim / 16;
    const Seq s = seq_at(c, b);
    const int p = s.p0 + t - s.q0;
    const bool known = p >= 0 && p < rope_rows;  // a position that the rotation table holds
    const int64_t slot = known && b < c.batch && p < c.cap ? slot_of(c, b, p) : -1;
    const uint16_t *src = qkv + t * ld;
    for (int u = threadIdx.x; u < (n_heads + 2 * c.n_kv) * per; u += kAppendThreads) {
        const int head = u / per, i = (u % per) * 8, kvh = (head - n_heads) % c.n_kv;
        const uint16_t *x = src + head * head_dim + i;
        uint16_t *dst = qo + (static_cast<int64_t>(t) * n_heads + head) * head_dim + i;
        if (head >= n_heads) {
            if (slot < 0) continue;
            dst = (head < n_heads + c.n_kv ? c.k : c.v) + slot + kvh * c.head_stride + i;
        }
        u32x4_t lo = *reinterpret_cast<const u32x4_t *>(x);
        u32x4_t hi = *reinterpret_cast<const u32x4_t *>(x + half);
        if (!known) {
            lo = hi = (u32x4_t){0, 0, 0, 0};
        } else if (head < n_heads + c.n_kv) {
            float a[8], d[8], ra[8], rd[8];
            unpack8<DT>(lo, a);
            unpack8<DT>(hi, d);
            const float4_t *cp = reinterpret_cast<const float4_t *>(cs + static_cast<int64_t>(p) * half + i);
            const float4_t *sp = reinterpret_cast<const float4_t *>(sn + static_cast<int64_t>(p) * half + i);
            const float4_t c0 = cp[0], c1 = cp[1], s0 = sp[0], s1 = sp[1];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float cj = j < 4 ? c0[j & 3] : c1[j & 3], sj = j < 4 ? s0[j & 3] : s1[j & 3];
                ra[j] = a[j] * cj - d[j] * sj;
                rd[j] = d[j] * cj + a[j] * sj;
            }
            lo = pack8<DT>(ra);
            hi = pack8<DT>(rd);
        }
        *reinterpret_cast<u32x4_t *>(dst) = lo;
        *reinterpret_cast<u32x4_t *>(dst + half) = hi;
    }
}

// ---------------------------------------------------------------------------- attention
//
// Rows.  The n_heads / n_kv query heads that share a key/value head, times a sequence's new
// tokens, are the rows of one product with that head's keys: row r is token r / group, head
// r % group.  Both kernels form S^T = K Q^T and O^T = V^T P^T, so that a lane holds scores and
// outputs of one row only (a column of the MFMA result): the softmax's maximum and sum stay in
// the lane, and the scores leave the first product in the register layout that the second one
// takes as its operand.
//
// Parts.  A sequence's positions [shared, end) are read through its own table row, [0, shared)
// through row 0 for the rows of the whole batch.  Both are cut into pieces where there are too
// few rows to fill the card; what a piece leaves is (maximum, sum, unscaled output) in fp32 for
// paged_attn_join_kernel, and the output itself where the piece is all there is of a row.

struct Query {
    const uint16_t *q;
    int64_t ld_tok, ld_head;
    uint16_t *out;
    float *lse;
    float *part_o;    // tiled parts: [tokens * n_heads][dense][D]
    float2 *part_ml;  // [tokens * n_heads][dense]
    int dense;        // pieces of the tiled parts; 0: their rows are written to `out`
    int n_heads, group, window, sinks, shared;
    float scale;      // of the scores in units of log 2, positive
    uint32_t flip;    // sign bits of a query pair, where the scale is negative
};

struct Part {       // a tiled part
    int prefix;     // 1: positions below `shared`, the whole batch's rows
    int splits;     // pieces of this part
    int first;      // index of its first piece
    int min_tiles;  // tiles of a piece, at least
    int blocks;     // row blocks
    int groups;     // workgroups
};

struct Few {         // the parts of few rows
    float *part_o;   // [slots * n_kv][rows of an item][D]
    float2 *part_ml; // [slots * n_kv][rows of an item]
    int2 *where;     // [1 + prefix][tokens * group]: (first slot, pieces * 64 + row in the item)
    int slots;       // all of them
    int groups;      // workgroups a key/value head
    int min_units;   // work of one, at least
    int whole;       // 1: an item each
    int items;       // at most
    int seqs, prefix; // entries: sequences, and 1 for the prefix if it has few rows
    int direct;      // 1: an item in one piece is written to `out`
};

constexpr int kNowhere = -(1 << 30);  // the position of a row that is not there

// A window of 64 pages of a sequence, a lane each, and the next 64 entries on their way: a page's
// offset is then a lane read away, where a scalar load of each entry would be waited for together
// with the LDS reads.
struct Pages {
    int64_t off;   // lane l: byte offset of page first + l, or -1 where the entry names no page
    int next;      // entry first + 64 + l
    int first;

    __device__ __forceinline__ int entry(const Cache &c, const int32_t *tab, int i) const {
        return i < (c.cap >> c.page_shift) ? tab[i] : -1;
    }
    __device__ __forceinline__ void set(const Cache &c, int e) {
        off = static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages) ? e * c.page_stride * 2 : -1;
    }
    __device__ __forceinline__ void begin() { first = -(1 << 30); }
    // the window that holds `page` (the wave's); windows begin where they are first asked for
    __device__ __forceinline__ void hold(const Cache &c, const int32_t *tab, int page) {
        if (page >= first && page < first + 64) return;
        const int l = threadIdx.x & 63;
        if (page >= first + 64 && page < first + 128) {
            first += 64;
            set(c, next);
        } else {
            first = page;
            set(c, entry(c, tab, first + l));
        }
        next = entry(c, tab, first + 64 + l);
    }
    // a page of the window, in keys or values of a head (`base`), as a buffer resource: one that
    // is not there, or not wanted, is an empty one, from which every load gives zeros
    __device__ __forceinline__ rsrc_t rsrc(const Cache &c, const uint16_t *base, bool want, int page,
                                           int row_bytes, bool &there) const {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(off), page - first);
        const int hi = __builtin_amdgcn_readlane(static_cast<int>(off >> 32), page - first);
        there = want && hi >= 0;
        const char *p = reinterpret_cast<const char *>(base) +
                        (there ? static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo) : 0);
        const int bytes = ((1 << c.page_shift) - 1) * static_cast<int>(c.slot_stride) * 2 + row_bytes;
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(p), static_cast<short>(0),
                                                 there ? bytes : 0, 0x00020000);
    }
    // byte of position k's slot in its page
    __device__ __forceinline__ static int slot(const Cache &c, int k) {
        return (k & ((1 << c.page_shift) - 1)) * static_cast<int>(c.slot_stride) * 2;
    }
};

// Loads of the few-rows kernel, not temporal (aux bit 1): a step reads its cache once, and lines
// that evict others on their way cost 2-4 % (131071 keys 60.6 -> 59.1 us, 64 sequences
// 212.7 -> 206.4 us).
__device__ __forceinline__ u32x4_t bload16s(rsrc_t r, int off, int soff) {
    return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, soff, 2));
}
__device__ __forceinline__ u32x2_t bload8s(rsrc_t r, int off, int soff) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(r, off, soff, 2));
}

// A row's probabilities are formed as 2^(score - m) and rounded to the 16-bit type for the second
// product; m lies kTop below the row's largest score, in units of log 2.  fp16 has 5 bits of
// exponent: with a largest of 1 a probability below 2^-14 loses bits and one below 2^-25 is gone,
// while the sum that divides them counts it (20000 keys 18 behind a first one whose value is 0,
// as behind a sink token: an output of zeros).  With a largest of 2^15 that begins at 2^-29.  The
// factor is in the sum as well, and by m in the joined rows and the log-sum-exp.
template <int DT>
constexpr float kTop = DT == NF4_BF16 ? 0.f : 15.f;

// The exponents are fma(score, scale, -m), exact but for their own rounding, with m the rounded
// score * scale of the largest: that one's exponent is what m's rounding left, and grows with m
// (16 and more from 2^28 on: past fp16's range).  From kFar on the products are rounded as m is
// and subtracted (two operations: the build contracts none), so that the largest's exponent is 0.
constexpr float kFar = 1 << 20;

// m of a row whose largest score * scale is t
template <int DT>
__device__ __forceinline__ float base_of(float t) {
    return fabsf(t) > kFar ? t : t - kTop<DT>;
}
// a score as its exponent at a base that is far (or -inf, of a row that saw nothing: as it is)
__device__ __forceinline__ float far_exponent(float score, float scale, float m) {
    return score * scale - (m == -INFINITY ? 0.f : m);
}
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > kFar && m != -INFINITY; }

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// A scalar load: table entries are the same for a wave.
__device__ __forceinline__ int sload(const int32_t *p) {
    return *(const __attribute__((address_space(4))) int32_t *)p;
}

// The position of token t, where the sequence differs from lane to lane.
__device__ __forceinline__ int position_of(const Cache &c, int t) {
    int b;
    if (c.cu) {
        int lo = 0, hi = c.batch;  // the first sequence that ends past t
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (c.cu[mid + 1] <= t) lo = mid + 1;
            else hi = mid;
        }
        b = lo;
    } else {
        b = t / c.uniform;
    }
    const Seq s = seq_at(c, b);
    return s.p0 + t - s.q0;
}

// The lowest n bits.
__device__ __forceinline__ uint64_t below(int n) {
    return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1;
}

// What a workgroup's rows (positions pmin .. pmax) see of a part: keys of [lo, hi) that are at
// most at the row's position, and past its window's start or below `sinks`; tiles of 2^SH keys,
// first those of the sinks, then those of the windows.
template <int SH>
struct Range {
    int lo, hi, pmin, pmax;
    int sink0, sinks_n, win0, n;  // tiles
    int i0, i1;                   // of this piece

    __device__ __forceinline__ void set(const Cache &c, const Query &a, int prefix) {
        const int end = pmax + 1 < c.cap ? pmax + 1 : c.cap;
        lo = prefix ? 0 : a.shared;
        hi = prefix && a.shared < end ? a.shared : end;
        int first = lo;
        if (a.window && pmin >= a.window && pmin - a.window + 1 > lo) first = pmin - a.window + 1;
        const int se = a.window ? (a.sinks < hi ? a.sinks : hi) : lo;
        n = 0;
        sinks_n = sink0 = win0 = 0;
        if (hi > lo) {
            sink0 = lo >> SH;
            win0 = first >> SH;
            const int s1 = se > lo ? (se + (1 << SH) - 1) >> SH : sink0, w1 = (hi + (1 << SH) - 1) >> SH;
            sinks_n = (s1 < win0 ? s1 : win0) - sink0;
            n = sinks_n + (w1 > win0 ? w1 - win0 : 0);
        }
        i0 = 0;
        i1 = n;
    }
    __device__ __forceinline__ void cut(int splits, int min_tiles, int piece) {
        int per = (n + splits - 1) / splits;
        per = per > min_tiles ? per : min_tiles;
        i0 = piece * per < n ? piece * per : n;
        i1 = i0 + per < n ? i0 + per : n;
    }
    __device__ __forceinline__ int key0(int i) const {
        return (i < sinks_n ? sink0 + i : win0 + i - sinks_n) << SH;
    }
    // every row sees every key of the tile at k (its pages apart)
    __device__ __forceinline__ bool full(const Query &a, int k) const {
        const int e = k + (1 << SH);
        return k >= lo && e <= hi && e <= pmin + 1 &&
               (!a.window || pmax - a.window < k || e <= a.sinks);
    }
    // some row sees key j
    __device__ __forceinline__ bool any(const Query &a, int j) const {
        return j >= lo && j < hi && (!a.window || pmin - a.window < j || j < a.sinks);
    }
    // the keys of the tile at k that some row sees, and that the row at position p sees, as bits
    // (a few instructions for a tile, where the tests below are a dozen for each key)
    __device__ __forceinline__ uint64_t any_bits(const Query &a, int k) const {
        uint64_t m = below(hi - k) & ~below(lo - k);
        if (a.window) m &= ~below(pmin - k - a.window + 1) | below(a.sinks - k);
        return m;
    }
    __device__ __forceinline__ uint64_t seen_bits(const Query &a, int p, int k) const {
        uint64_t m = below((hi < p + 1 ? hi : p + 1) - k) & ~below(lo - k);
        if (a.window) m &= ~below(p - k - a.window + 1) | below(a.sinks - k);
        return m;
    }
    // the row at position p sees key j
    __device__ __forceinline__ bool sees(const Query &a, int p, int j) const {
        return j >= lo && j < hi && j <= p && (!a.window || p - a.window < j || j < a.sinks);
    }
};

// 16-bit pairs that hold an infinity or a NaN.
template <int DT>
__device__ __forceinline__ bool not_finite(uint32_t w) {
    constexpr uint32_t e = DT == NF4_BF16 ? 0x7f80u : 0x7c00u;
    return (w & e) == e || ((w >> 16) & e) == e;
}

// 0 where all 8 values of a chunk are finite, else NaN; added to `c`.
template <int DT>
__device__ __forceinline__ float odd_sum(const u32x4_t &r, float c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = dot2<DT>(r[i], 0, c);
    return c;
}

template <int DT>
__device__ __forceinline__ uint32_t finite_or_zero(uint32_t w) {
    constexpr uint32_t e = DT == NF4_BF16 ? 0x7f80u : 0x7c00u;
    return ((w & e) == e ? 0u : w & 0xffffu) | (((w >> 16) & e) == e ? 0u : w & 0xffff0000u);
}

// The value of 16 bits where it is an infinity or a NaN, else 0.
template <int DT>
__device__ __forceinline__ float odd_part(uint32_t h) {
    return not_finite<DT>(h & 0xffffu) ? f32_of<DT>(h & 0xffffu) : 0.f;
}

template <int DT>
__device__ __forceinline__ float4_t mfma16(const u32x4_t &a, const u32x4_t &b, const float4_t &c) {
    if constexpr (DT == NF4_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf168_t, a),
                                                      __builtin_bit_cast(bf168_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a),
                                                     __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// Two outputs.  An output is a mean of values, so one past fp16's last number is there by the
// roundings of its probabilities (at most one step), and is that number; an infinity that is among
// the values stays.
template <int DT>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
    if constexpr (DT == NF4_F16) {
        constexpr float most = 65504.f;
        a = fabsf(a) < INFINITY ? __builtin_amdgcn_fmed3f(a, -most, most) : a;
        b = fabsf(b) < INFINITY ? __builtin_amdgcn_fmed3f(b, -most, most) : b;
    }
    return pack2<DT>(a, b);
}

// 8 consecutive values of a query row, its sign as the scale's.
__device__ __forceinline__ u32x4_t load_q(const Query &a, int tok, int head, int d) {
    u32x4_t r = *reinterpret_cast<const u32x4_t *>(a.q + tok * a.ld_tok + head * a.ld_head + d);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] ^= a.flip;
    return r;
}

// ------------------------------------------------------------- few rows (decoding)
//
// Work.  An item is at most 16 RB rows of a sequence (more are further items) and all that they
// see; it costs a unit to begin and one for every step, a slab of 32 keys for each of the
// workgroup's W waves.  Lengths are known on the device only, so every workgroup adds up all
// sequences' units (64 at a time, a lane each) and takes an equal share of the total, which ends
// and begins inside items: all workgroups are resident and finish together, however uneven the
// lengths (a fixed number of pieces per sequence instead: 64 sequences of 40 to 16000 keys
// 399 us).  A piece's slot is its workgroup's number plus its item's: two pieces of one
// workgroup, or two workgroups in one item, never have the same.

template <int D>
constexpr int few_lds(int waves, int rb) { return waves * 16 * rb * ((D + 4) * 4 + 8); }

struct Units {
    int64_t total, base, up;   // units: of all entries; before this chunk; to this lane's end
    int ibase, iup;            // items, alike
    int b0, steps, blocks;     // first entry of the chunk; this lane's entry
    int pmin, pmax;            // positions of the whole batch (if a prefix is an entry)
};

// `div` of an equal cut: the first unit of workgroup g of n
__device__ __forceinline__ int64_t first_unit(int64_t total, int g, int n) {
    const uint64_t x = static_cast<uint64_t>(g) * static_cast<uint64_t>(total);
    if (x >> 32) return static_cast<int64_t>(x / static_cast<uint32_t>(n));
    return static_cast<uint32_t>(x) / static_cast<uint32_t>(n);
}

// the workgroup whose share holds unit u: the largest g with g total < (u + 1) n
__device__ __forceinline__ int group_of(int64_t total, int64_t u, int n) {
    const uint64_t x = static_cast<uint64_t>(u + 1) * static_cast<uint32_t>(n) - 1;
    if ((x | static_cast<uint64_t>(total)) >> 32) return static_cast<int>(x / static_cast<uint64_t>(total));
    return static_cast<uint32_t>(x) / static_cast<uint32_t>(total);
}

__device__ __forceinline__ int groups_used(const Few &f, int64_t total) {
    const int64_t n = total / f.min_units;
    return n < 1 ? 1 : n < f.groups ? static_cast<int>(n) : f.groups;
}

template <int W, int RB>
__device__ __forceinline__ void load_units(Units &u, const Cache &c, const Query &a, const Few &f,
                                           int b0) {
    const int l = threadIdx.x & 63, e = b0 + l;
    u.b0 = b0;
    u.steps = u.blocks = 0;
    if (e < f.seqs + f.prefix) {
        Range<5> rg;
        int rows = c.tokens * a.group;
        rg.pmin = u.pmin;
        rg.pmax = u.pmax;
        if (e < f.seqs) {
            const Seq s = seq_at(c, e);
            rows = s.n * a.group;
            rg.pmin = s.p0;
            rg.pmax = s.p0 + s.n - 1;
        }
        rg.set(c, a, e == f.seqs);
        u.blocks = (rows + 16 * RB - 1) / (16 * RB);
        u.steps = (rg.n + W - 1) / W;
    }
    u.up = static_cast<int64_t>(u.blocks) * (f.whole ? 1 : u.steps + 1);
    u.iup = u.blocks;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t x = __shfl_up(u.up, o);
        const int y = __shfl_up(u.iup, o);
        if (l >= o) {
            u.up += x;
            u.iup += y;
        }
    }
}

__device__ __forceinline__ int64_t last_lane(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), 63);
    const int hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), 63);
    return (static_cast<int64_t>(hi) << 32) | lo;
}

__device__ __forceinline__ int64_t lane_of(int64_t v, int l) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), l);
    const int hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), l);
    return (static_cast<int64_t>(hi) << 32) | lo;
}

// The total, and the chunk of the first 64 entries.
template <int W, int RB>
__device__ __forceinline__ void all_units(Units &u, const Cache &c, const Query &a, const Few &f) {
    u.pmin = 0x7fffffff;
    u.pmax = kNowhere;
    if (f.prefix) {
        for (int b0 = 0; b0 < f.seqs; b0 += 64) {
            const int e = b0 + (threadIdx.x & 63);
            if (e >= f.seqs) continue;
            const Seq s = seq_at(c, e);
            if (s.n == 0) continue;
            u.pmin = s.p0 < u.pmin ? s.p0 : u.pmin;
            u.pmax = s.p0 + s.n - 1 > u.pmax ? s.p0 + s.n - 1 : u.pmax;
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_xor(u.pmin, o), z = __shfl_xor(u.pmax, o);
            u.pmin = x < u.pmin ? x : u.pmin;
            u.pmax = z > u.pmax ? z : u.pmax;
        }
        u.pmin = __builtin_amdgcn_readfirstlane(u.pmin);
        u.pmax = __builtin_amdgcn_readfirstlane(u.pmax);
    }
    u.total = u.base = 0;
    u.ibase = 0;
    const int n = f.seqs + f.prefix;
    for (int b0 = 0; b0 < n; b0 += 64) {
        load_units<W, RB>(u, c, a, f, b0);
        u.total += last_lane(u.up);
    }
    if (n > 64) load_units<W, RB>(u, c, a, f, 0);
}

template <int W, int RB>
__device__ __forceinline__ void next_units(Units &u, const Cache &c, const Query &a, const Few &f) {
    u.base += last_lane(u.up);
    u.ibase += __builtin_amdgcn_readlane(u.iup, 63);
    load_units<W, RB>(u, c, a, f, u.b0 + 64);
}

// The bytes of the cache are all that counts, and no key is used often enough for LDS to pay.
// Each wave takes every W-th 32-key slab on its own, straight from memory into MFMA operands: a
// lane loads 16 bytes of a key (rows of K are A-operand rows as they lie) and 16 bytes (8
// channels) of 8 of its V rows, and turns the 8x8 block of V into operands by byte permutes,
// which is free beside the memory (channel e of each lane's 8 forms one product, so the order of
// channels is a permuted one).  The next slab's keys are loaded as soon as the scores are formed
// and its values as soon as they are used, so that a wave always has loads in flight; the waves'
// results meet in LDS.

//
// Bound by memory.  bf16, 4 heads of 128: 64 ragged sequences, 1.14 GB, in 199 us (5.7 TB/s, where
// a plain read of this card reaches 5.6); 131071 keys of one, 268 MB, in 51.5 us (5.2 TB/s) and 5 us
// for the join.  Up to kWholeKeys keys of a sequence it is latency: length, page entries, keys,
// the sums over LDS, 9.4 us.  (SMALL: an address a lane, for pages under 16 slots and pages whose
// slots span 2^31 bytes.)

template <int DT, int D, int RB, bool SMALL, int W>
__device__ __forceinline__ void few_body(const Cache &c, const Query &a, const Few &f, int block,
                                         uint8_t *lds) {
    constexpr int KC = D / 32, VE = D / 16, LD = D + 4;  // K chunks, V values a lane, LDS row
    float *s_o = reinterpret_cast<float *>(lds);                           // [W][16 RB][LD]
    float2 *s_ml = reinterpret_cast<float2 *>(s_o + W * 16 * RB * LD);     // [W][16 RB]
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
    const int g = l >> 4, n = l & 15;
    const int kvh = block % c.n_kv, group = block / c.n_kv;
    const uint16_t *kb = c.k + kvh * c.head_stride, *vb = c.v + kvh * c.head_stride;
    const int stride2 = static_cast<int>(c.slot_stride) * 2;
    const int page_mask = (1 << c.page_shift) - 1;

    Units u;
    int used = 0;
    int64_t at = group, u1 = group + 1;
    const bool plain = W == 8 && !c.cu;  // whole sequences of at most 16 rows: item b is sequence b
    if (plain) {
        if (group >= f.seqs) return;
    } else {
        all_units<W, RB>(u, c, a, f);
        used = f.whole ? 0 : groups_used(f, u.total);
        if (f.whole ? group >= u.total : group >= used) return;
        if (!f.whole) {
            u1 = first_unit(u.total, group + 1, used);
            at = first_unit(u.total, group, used);
        }
    }
    while (at < u1) {
        // the item that unit `at` falls into
        int b = group, item = group, blk = 0, st0 = 0, st1 = 0, steps = 0, pieces = 1;
        bool single = true;
        if (!plain) {
            uint64_t past = __ballot(u.base + u.up > at);
            while (!past) {
                if (u.b0 + 64 >= f.seqs + f.prefix) return;  // lengths that changed under the kernel
                next_units<W, RB>(u, c, a, f);
                past = __ballot(u.base + u.up > at);
            }
            const int lane = __builtin_ctzll(past);
            b = u.b0 + lane;
            steps = __builtin_amdgcn_readlane(u.steps, lane);
            const int blocks = __builtin_amdgcn_readlane(u.blocks, lane);
            const int per = f.whole ? 1 : steps + 1;
            int64_t start = u.base + lane_of(u.up, lane) - static_cast<int64_t>(blocks) * per;
            blk = blocks == 1 ? 0 : static_cast<int>((at - start) / per);
            start += static_cast<int64_t>(blk) * per;
            item = u.ibase + __builtin_amdgcn_readlane(u.iup, lane) - blocks + blk;
            const int64_t next = start + per < u1 ? start + per : u1;
            st0 = static_cast<int>(at - start) - 1;
            st1 = f.whole ? steps : static_cast<int>(next - start) - 1;
            st0 = st0 < 0 ? 0 : st0;
            at = next;
            if (item >= f.items) return;        // offsets that decrease
            if (st1 <= st0 && steps) continue;  // no more than its beginning
            single = st0 == 0 && st1 == steps;
            if (!single && st0 == 0) pieces = group_of(u.total, start + steps, used) - group + 1;
        } else {
            at = u1;
        }

        const bool prefix = b == f.seqs;
        Seq s = {0, c.tokens, 0};
        if (!prefix) s = seq_uniform(c, b);
        const int rows = s.n * a.group, r0 = blk * 16 * RB;
        const int32_t *tab = c.table + (prefix ? 0 : b) * c.ld_table;
        // this lane's rows and their positions
        u32x4_t q[RB][KC];
        int pos[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = r0 + rb * 16 + n;
            pos[rb] = kNowhere;
#pragma unroll
            for (int k = 0; k < KC; ++k) q[rb][k] = (u32x4_t){0, 0, 0, 0};
            if (r < rows) {
                const int tok = s.q0 + r / a.group, head = kvh * a.group + r % a.group;
                pos[rb] = prefix ? position_of(c, tok) : s.p0 + r / a.group;
#pragma unroll
                for (int k = 0; k < KC; ++k) q[rb][k] = load_q(a, tok, head, k * 32 + g * 8);
            }
        }
        Range<5> rg;  // of all the entry's rows, as its steps were counted
        rg.pmin = prefix ? u.pmin : s.p0;
        rg.pmax = prefix ? u.pmax : s.p0 + s.n - 1;
        rg.set(c, a, prefix);
        if (!plain) {
            rg.i0 = st0 * W;
            rg.i1 = st1 * W < rg.n ? st1 * W : rg.n;
        }

        float m[RB], sum[RB];
        bool far[RB];  // a row's m is far (the wave's)
        float4_t acc[RB][VE];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            m[rb] = -INFINITY;
            far[rb] = false;
            sum[rb] = 0.f;
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[rb][e] = (float4_t){0.f, 0.f, 0.f, 0.f};
        }

        // pages under 16 slots (SMALL): the entry of key k + l % 32; none past the item's end
        auto entry = [&](int i, int k) {
            const int j = k + (l & 31);
            return i < rg.i1 && j < c.cap ? tab[j >> c.page_shift] : -1;
        };
        auto good = [&](int e) { return static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages); };
        u32x4_t kr[2][KC];
        u32x4_t vr[8];
        Pages pg;
        pg.begin();
        // Every load is issued, whether its page is there or not: the waits then are exact.
        // Returns the slab's keys whose page is there.
        auto load_k = [&](int i, int k, int e) -> uint32_t {
            uint32_t ok = 0;
            if constexpr (SMALL) {
                ok = static_cast<uint32_t>(__ballot(good(e)));
            } else if (i < rg.i1) {
                pg.hold(c, tab, k >> c.page_shift);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (SMALL) {
                    const int eh = __shfl(e, h * 16 + n);
                    const uint16_t *p = kb + (good(eh) ? eh * c.page_stride + ((k + h * 16 + n) & page_mask) * c.slot_stride : 0);
#pragma unroll
                    for (int x = 0; x < KC; ++x) {
                        kr[h][x] = (u32x4_t){0, 0, 0, 0};
                        if (good(eh)) kr[h][x] = *reinterpret_cast<const u32x4_t *>(p + g * 8 + x * 32);
                    }
                } else {
                    const int kh = k + h * 16;
                    bool there;
                    const rsrc_t r = pg.rsrc(c, kb, i < rg.i1, kh >> c.page_shift, D * 2, there);
                    ok |= there ? 0xffffu << (16 * h) : 0;
                    const int so = Pages::slot(c, kh);
#pragma unroll
                    for (int x = 0; x < KC; ++x) kr[h][x] = bload16s(r, n * stride2 + g * 16 + x * 64, so);
                }
            }
            return ok;
        };
        auto load_v = [&](int i, int k, int e) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                rsrc_t r;
                int so = 0;
                if constexpr (!SMALL) {
                    bool there;
                    r = pg.rsrc(c, vb, i < rg.i1, (k + h * 16) >> c.page_shift, D * 2, there);
                    so = Pages::slot(c, k + h * 16);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (SMALL) {
                        const int i = h * 16 + g * 4 + j, eh = __shfl(e, i);
                        vr[h * 4 + j] = (u32x4_t){0, 0, 0, 0};
                        if (good(eh)) {
                            const u32x2_t *p = reinterpret_cast<const u32x2_t *>(
                                vb + eh * c.page_stride + ((k + i) & page_mask) * c.slot_stride + n * VE);
                            const u32x2_t lo = p[0], hi = p[D == 128 ? 1 : 0];
                            vr[h * 4 + j] = (u32x4_t){lo.x, lo.y, hi.x, hi.y};
                        }
                    } else if constexpr (D == 128) {
                        vr[h * 4 + j] = bload16s(r, (g * 4 + j) * stride2 + n * 16, so);
                    } else {
                        const u32x2_t t = bload8s(r, (g * 4 + j) * stride2 + n * 8, so);
                        vr[h * 4 + j] = (u32x4_t){t.x, t.y, 0, 0};
                    }
                }
            }
        };

        bool odd_seen = false;
        int i = rg.i0 + w, k = rg.key0(i), k2 = rg.key0(i + W), e0 = -1, e1 = -1;
        uint32_t ok = 0;  // keys whose page is there
        if (i < rg.i1) {
            if constexpr (SMALL) {
                e0 = entry(i, k);
                e1 = entry(i + W, k2);
            }
            ok = load_k(i, k, e0);
            load_v(i, k, e0);
        }
        while (i < rg.i1) {
            float4_t st[RB][2];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    st[rb][h] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int x = 0; x < KC; ++x) st[rb][h] = mfma16<DT>(kr[h][x], q[rb][x], st[rb][h]);
                }
            const uint32_t ok2 = load_k(i + W, k2, e1);
            const bool full = rg.full(a, k) && ok == 0xffffffffu;
            bool odd = false;  // an infinity or NaN among values that not every row sees
            if (!full) {
                const uint32_t any = static_cast<uint32_t>(rg.any_bits(a, k)) & ok;
                float zero = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (!(((any >> (g * 4)) >> ((j >> 2) * 16 + (j & 3))) & 1)) vr[j] = (u32x4_t){0, 0, 0, 0};
                    zero = odd_sum<DT>(vr[j], zero);
                }
                odd = rg.pmin != rg.pmax && zero != 0.f;  // (rows of one token see the same keys)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const uint32_t see = (static_cast<uint32_t>(rg.seen_bits(a, pos[rb], k)) & ok) >> (g * 4);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (!((see >> ((j >> 2) * 16 + (j & 3))) & 1)) st[rb][j >> 2][j & 3] = -INFINITY;
                }
            }
            u32x4_t pf[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float top = st[rb][0][0];
#pragma unroll
                for (int j = 1; j < 8; ++j) top = fmaxf(top, st[rb][j >> 2][j & 3]);
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float mn = fmaxf(m[rb], base_of<DT>(top * a.scale));
                if (__any(mn > m[rb])) {
                    const float alpha = mn > m[rb] ? __builtin_amdgcn_exp2f(m[rb] - mn) : 1.f;
                    sum[rb] *= alpha;
#pragma unroll
                    for (int e = 0; e < VE; ++e) acc[rb][e] *= alpha;
                    m[rb] = mn;
                    far[rb] = __any(is_far(mn));
                }
                if (__builtin_expect(far[rb], 0)) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        st[rb][j >> 2][j & 3] = far_exponent(st[rb][j >> 2][j & 3], a.scale, m[rb]);
                }
                const float mul = far[rb] ? 1.f : a.scale;
                const float base = far[rb] || m[rb] == -INFINITY ? 0.f : m[rb];
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = __builtin_amdgcn_exp2f(fmaf(st[rb][j >> 2][j & 3], mul, -base));
                    sum[rb] += p[j];
                }
                // probabilities in the 16-bit type for the MFMA (two products of halves would take
                // twice the instructions); their sum stays unrounded
                pf[rb] = (u32x4_t){pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]),
                                   pack2<DT>(p[4], p[5]), pack2<DT>(p[6], p[7])};
            }
            if (__any(odd)) {
                // 0 times such a value is no 0: zeros take their place, below they are added to
                // the rows that see them
                odd_seen = true;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int x = 0; x < VE / 2; ++x) vr[j][x] = finite_or_zero<DT>(vr[j][x]);
            }
#pragma unroll
            for (int e = 0; e < VE; ++e) {  // operand of channel e: half e & 1 of word e / 2 of 8 rows
                const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
                u32x4_t f;
#pragma unroll
                for (int x = 0; x < 4; ++x) f[x] = vperm(vr[2 * x + 1][e >> 1], vr[2 * x][e >> 1], sel);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) acc[rb][e] = mfma16<DT>(f, pf[rb], acc[rb][e]);
            }
            load_v(i + W, k2, e1);
            ok = ok2;
            i += W;
            k = k2;
            k2 = rg.key0(i + W);
            if constexpr (SMALL) {
                e0 = e1;
                e1 = entry(i + W, k2);
            }
        }

        if (odd_seen) {
            // infinities and NaN among values that not every row sees: a probability above 0
            // leaves them what they are
#pragma unroll 1
            for (i = rg.i0 + w; i < rg.i1; i += W) {
                k = rg.key0(i);
                // (full slabs, as above: their products have them already)
                if (rg.full(a, k) && !~__ballot(good(tab[(k + (l & 31)) >> c.page_shift]))) continue;
#pragma unroll 1
                for (int key = k; key < k + 32; ++key) {
                    if (!rg.any(a, key)) continue;
                    const int e = sload(tab + (key >> c.page_shift));
                    if (!good(e)) continue;
                    const uint16_t *p = vb + e * c.page_stride + (key & page_mask) * c.slot_stride;
#pragma unroll
                    for (int x = 0; x < 4; ++x)
#pragma unroll
                        for (int z = 0; z < VE; ++z) {
                            const float o = odd_part<DT>(p[(g * 4 + x) * VE + z]);
#pragma unroll
                            for (int rb = 0; rb < RB; ++rb)
                                acc[rb][z][x] += rg.sees(a, pos[rb], key) ? o : 0.f;
                        }
                }
            }
        }

        // the waves' parts: each scaled to the common maximum, summed over LDS in wave order
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            sum[rb] += __shfl_xor(sum[rb], 16);
            sum[rb] += __shfl_xor(sum[rb], 32);
            if (m[rb] == -INFINITY && sum[rb] != sum[rb]) m[rb] = 0.f;  // NaN scores only: not nothing
            const int row = w * 16 * RB + rb * 16 + n;
            if (g == 0) s_ml[row] = make_float2(m[rb], sum[rb]);
            if (r0 + rb * 16 + n < rows) {
#pragma unroll
                for (int x = 0; x < 4; ++x)
#pragma unroll
                    for (int e = 0; e < VE; e += 4)
                        *reinterpret_cast<float4_t *>(s_o + row * LD + (g * 4 + x) * VE + e) =
                            (float4_t){acc[rb][e][x], acc[rb][e + 1][x], acc[rb][e + 2][x],
                                       acc[rb][e + 3][x]};
            }
        }
        __syncthreads();
        for (int v = threadIdx.x; v < 16 * RB * (D / 4); v += W * 64) {
            const int r = v / (D / 4), d = (v % (D / 4)) * 4;
            if (r0 + r >= rows) continue;
            float mm = -INFINITY, ll = 0.f;
            float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < W; ++x) mm = fmaxf(mm, s_ml[x * 16 * RB + r].x);
#pragma unroll
            for (int x = 0; x < W; ++x) {
                const float2 ml = s_ml[x * 16 * RB + r];
                const float fx = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - mm);
                ll += ml.y * fx;
                o += *reinterpret_cast<const float4_t *>(s_o + (x * 16 * RB + r) * LD + d) * fx;
            }
            if (single && f.direct) {
                const int64_t row = static_cast<int64_t>(s.q0 + (r0 + r) / a.group) * a.n_heads +
                                    kvh * a.group + (r0 + r) % a.group;
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                *reinterpret_cast<u32x2_t *>(a.out + row * D + d) =
                    (u32x2_t){pack_out<DT>(o[0] * inv, o[1] * inv), pack_out<DT>(o[2] * inv, o[3] * inv)};
                if (a.lse && d == 0) a.lse[row] = ll == 0.f ? -INFINITY : mm * kLn2 + logf(ll);
            } else {
                const int64_t slot = (static_cast<int64_t>(group + item) * c.n_kv + kvh) * 16 * RB + r;
                if (mm != -INFINITY) *reinterpret_cast<float4_t *>(f.part_o + slot * D + d) = o;
                if (d == 0) f.part_ml[slot] = make_float2(mm, ll);
            }
        }
        if (W != 8 && kvh == 0 && st0 == 0) {  // the item's first piece says where its rows are
            const int r = threadIdx.x;
            if (r < 16 * RB && r0 + r < rows)
                f.where[(prefix ? c.tokens * a.group : 0) + s.q0 * a.group + r0 + r] =
                    make_int2(group + item, pieces * 64 + r);
        }
        __syncthreads();
    }
}

template <int DT, int D, int RB, bool SMALL, int W>
__global__ __launch_bounds__(64 * W, RB > 2 ? 1 : 2) void paged_attn_few_kernel(
    const Cache c, const Query a, const Few f) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[few_lds<D>(W, RB)];
    few_body<DT, D, RB, SMALL, W>(c, a, f, blockIdx.x, lds);
}

// ------------------------------------------------------------------ many rows (prompts)
//
// 128 rows a workgroup, 32 a wave on v_mfma_f32_32x32x16, over 64-key tiles: K and V tiles go to
// LDS by DMA while the tile before is used (two stages, one barrier a tile; two workgroups a CU).
// 16-byte chunk ch of K's row r lies at chunk ch ^ (r & 15) (128 channels; 64: ch ^ (r / 2 & 7)):
// the 16 lanes that LDS serves at a time then read 16 rows from 16 different bank groups.  V is
// read transposed (ds_read_b64_tr_b16: 4 keys of a channel a lane) from rows whose 64-byte blocks
// are exchanged by the key's low bits, 4 keys x 64 bytes on all banks.  No bank conflicts counted.
//
// 8192 new tokens, 28 heads of 128 over 4, bf16: 500-531 us from card to card, 906-962 TFLOP/s,
// where a library's 8192^3 product reaches 1130.  The matrix pipe is in use 42 % of the cycles,
// and the clock falls to 1.9 GHz under the load: the power cap bounds it.  64-wide heads: 174 us,
// 690 TFLOP/s, half the products for the same exponentials.  Measured against it (when it kept its
// maximum 2^8 behind and took 495): the next tile's scores formed beside this one's exponentials
// within a wave (fewer cycles, a lower clock: 495 us, and 5-15 % slower with few tiles), the same
// with 256 rows a workgroup (510 us).

typedef short v4i16_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16_t lds_v4i16_t;

// the value of lane l ^ 32
__device__ __forceinline__ float other_half(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

// by LDS address
__device__ __forceinline__ u32x2_t tr_read(uint32_t at) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        reinterpret_cast<lds_v4i16_t *>(static_cast<uintptr_t>(at))));
}
__device__ __forceinline__ u32x4_t lds16(uint32_t at) {
    return *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t *>(static_cast<uintptr_t>(at));
}

constexpr int kRows = 128;

template <int D>
constexpr int kTileLds = 4 * 64 * D * 2 + 64;  // two stages of K and V, and a few words

template <int DT, int D, bool SMALL>
__device__ __forceinline__ void tile_body(const Cache &c, const Query &a, const Part &part, int block,
                                          uint8_t *lds) {
    constexpr int CH = D / 8, KS = D / 16, DT32 = D / 32;  // 16-byte chunks of a row, k steps, d tiles
    constexpr int RPP = 256 / CH, PASS = 64 / RPP;         // rows a pass of the workgroup loads
    constexpr int STAGE = 64 * D * 2;
    uint8_t *s_k = lds, *s_v = lds + 2 * STAGE;                // [2][STAGE]
    int *s_odd = reinterpret_cast<int *>(lds + 4 * STAGE);  // [2]: the stage's tile, where its
                                                            // values hold an infinity or NaN
    int *s_p = s_odd + 4;                                   // [8]
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63;
    const int g = l >> 5, n = l & 31;
    const int kvh = block % c.n_kv, y = block / c.n_kv;
    const int piece = y % part.splits;
    int blk = y / part.splits, b = 0;
    Seq s = {0, c.tokens, 0};
    if (!part.prefix) {
        blk = part.blocks - 1 - blk;  // the last rows see most: first
        // the sequence that row block blk falls into, 64 sequences at a time (the one past the
        // last holds the tokens past the last offset)
        for (b = 0;; b += 64) {
            if (b > c.batch) return;
            int nb = 0;
            if (b + l <= c.batch) nb = (seq_at(c, b + l).n * a.group + kRows - 1) / kRows;
            int upto = nb;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(upto, o);
                if (l >= o) upto += x;
            }
            const uint64_t past = __ballot(upto > blk);
            if (past) {
                const int f = __builtin_ctzll(past);
                blk -= __builtin_amdgcn_readlane(upto - nb, f);
                b += f;
                break;
            }
            blk -= __builtin_amdgcn_readlane(upto, 63);
        }
        s = seq_uniform(c, b);
    }
    const uint16_t *kb = c.k + kvh * c.head_stride, *vb = c.v + kvh * c.head_stride;
    const int stride2 = static_cast<int>(c.slot_stride) * 2;
    const int r0 = blk * kRows, rows = s.n * a.group;
    const int32_t *tab = c.table + b * c.ld_table;
    const int page_mask = (1 << c.page_shift) - 1;

    // this lane's row
    const int r = r0 + w * 32 + n;
    const bool live = r < rows;
    const int tok = s.q0 + (live ? r / a.group : 0), head = kvh * a.group + (live ? r % a.group : 0);
    int pos = kNowhere;
    if (live) pos = part.prefix ? position_of(c, tok) : s.p0 + r / a.group;
    u32x4_t q[KS];
#pragma unroll
    for (int x = 0; x < KS; ++x) {
        q[x] = (u32x4_t){0, 0, 0, 0};
        if (live) q[x] = load_q(a, tok, head, x * 16 + g * 8);
    }
    Range<6> rg;
    if (part.prefix) {
        int lo = live ? pos : 0x7fffffff, hi = pos;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_xor(lo, o), z = __shfl_xor(hi, o);
            lo = x < lo ? x : lo;
            hi = z > hi ? z : hi;
        }
        if (l == 0) {
            s_p[w] = lo;
            s_p[4 + w] = hi;
        }
        __syncthreads();
        for (int x = 0; x < 4; ++x) {
            lo = s_p[x] < lo ? s_p[x] : lo;
            hi = s_p[4 + x] > hi ? s_p[4 + x] : hi;
        }
        rg.pmin = __builtin_amdgcn_readfirstlane(lo);
        rg.pmax = __builtin_amdgcn_readfirstlane(hi);
    } else {
        const int last = r0 + kRows < rows ? r0 + kRows : rows;
        rg.pmin = s.p0 + r0 / a.group;
        rg.pmax = s.p0 + (last - 1) / a.group;
    }
    rg.set(c, a, part.prefix);
    rg.cut(part.splits, part.min_tiles, piece);

    float m = -INFINITY, sum = 0.f;
    bool odd_seen = false, far = false;  // far: a row's m is (the wave's)
    float16_t acc[DT32];
#pragma unroll
    for (int x = 0; x < DT32; ++x) acc[x] = (float16_t){};

    // ---- staging: a thread's row of a pass and its 16 bytes of it in LDS, and the chunk of the
    // row that belongs there
    const int srow = tid / CH, sch = tid % CH;
    const int kch = sch ^ (D == 128 ? srow & 15 : (srow >> 1) & 7);
    const int vch0 = sch ^ (D == 128 ? (srow & 3) << 2 : ((srow >> 1) & 1) << 2);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
                              (__attribute__((address_space(3))) uint8_t *)lds)) + w * 1024;
    auto good = [&](int e) { return static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages); };
    Pages pg;
    pg.begin();
    const int ko = (srow & 15) * stride2 + kch * 16, vo = (srow & 15) * stride2 + vch0 * 16;
    // tile k into stage st, and which of its keys' pages are there: by DMA, a pass of a wave
    // within one of the tile's 16-key quarters
    auto send = [&](int st, int k) -> uint64_t {
        uint64_t ok = 0;
        if constexpr (SMALL) {
            const int mine = k + l < c.cap ? tab[(k + l) >> c.page_shift] : -1;
            ok = __ballot(good(mine));
#pragma unroll
            for (int x = 0; x < PASS; ++x) {
                const int row = x * RPP + srow, e = __shfl(mine, row);
                const int64_t at = e * c.page_stride + ((k + row) & page_mask) * c.slot_stride;
                u32x4_t kx = {0, 0, 0, 0}, vx = {0, 0, 0, 0};
                if (good(e)) {
                    kx = *reinterpret_cast<const u32x4_t *>(kb + at + kch * 8);
                    vx = *reinterpret_cast<const u32x4_t *>(vb + at + vch0 * 8);
                }
                *reinterpret_cast<u32x4_t *>(s_k + st * STAGE + row * D * 2 + sch * 16) = kx;
                *reinterpret_cast<u32x4_t *>(s_v + st * STAGE + row * D * 2 + sch * 16) = vx;
            }
        } else {
            pg.hold(c, tab, k >> c.page_shift);
            if (c.page_shift >= 6) {  // the tile is in one page
                bool there;
                const int page = k >> c.page_shift, so = Pages::slot(c, k);
                const rsrc_t rk = pg.rsrc(c, kb, true, page, D * 2, there), rv = pg.rsrc(c, vb, true, page, D * 2, there);
                const uint32_t at = __builtin_amdgcn_readfirstlane(lds0 + st * STAGE);
                const int so1 = so + (D == 64 ? (w >> 1) * 16 : 0) * stride2;
#pragma unroll
                for (int x = 0; x < PASS; ++x) {
                    lds_dma16(at + x * 4096, ko, rk, so1 + x * RPP * stride2);
                    lds_dma16(at + 2 * STAGE + x * 4096, vo, rv, so1 + x * RPP * stride2);
                }
                return there ? ~0ull : 0;
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                bool there;
                const int k16 = k + x * 16, page = k16 >> c.page_shift;
                const rsrc_t rk = pg.rsrc(c, kb, true, page, D * 2, there), rv = pg.rsrc(c, vb, true, page, D * 2, there);
                ok |= there ? 0xffffull << (16 * x) : 0;
                if (D == 64 && (x & 1) != w >> 1) continue;
                const int so = Pages::slot(c, k16);
                const uint32_t at = __builtin_amdgcn_readfirstlane(lds0 + st * STAGE + (D == 128 ? x : x >> 1) * 4096);
                lds_dma16(at, ko, rk, so);
                lds_dma16(at + 2 * STAGE, vo, rv, so);
            }
        }
        return ok;
    };
    // what this wave loaded of a tile that not every row sees whole: the values of keys that no
    // row sees become zeros; infinities and NaN too (0 times one is no 0), and s_odd says so
    auto clean = [&](int st, int i, int k, uint64_t ok) {
        const uint64_t any = rg.any_bits(a, k) & ok;
        u32x4_t v[PASS];
        float zero = 0.f;
#pragma unroll
        for (int x = 0; x < PASS; ++x) {
            const int row = x * RPP + srow;
            u32x4_t *p = reinterpret_cast<u32x4_t *>(s_v + st * STAGE + row * D * 2 + sch * 16);
            v[x] = *p;
            if (!((any >> row) & 1)) *p = v[x] = (u32x4_t){0, 0, 0, 0};
            zero = odd_sum<DT>(v[x], zero);
        }
        if (zero != 0.f) {
#pragma unroll
            for (int x = 0; x < PASS; ++x) {
#pragma unroll
                for (int z = 0; z < 4; ++z) v[x][z] = finite_or_zero<DT>(v[x][z]);
                *reinterpret_cast<u32x4_t *>(s_v + st * STAGE + (x * RPP + srow) * D * 2 + sch * 16) = v[x];
            }
            s_odd[st] = i;
        }
    };

    // ---- operand addresses of this lane
    // (chunk numbers change by exclusive or: so do the addresses, whose low bits they are)
    const uint32_t lds_k = lds0 - w * 1024;
    const uint32_t kbase = lds_k + n * D * 2 + ((g ^ (D == 128 ? (n & 15) : ((n >> 1) & 7))) << 4);
    const int vkey = g * 4 + ((l & 15) >> 2);  // key (of 16) and chunk that it points at
    const int vch = ((l >> 4) & 1) * 2 + ((l & 3) >> 1);
    const uint32_t vbase = lds_k + 2 * STAGE + vkey * D * 2 + (l & 1) * 8 +
                           ((vch ^ (D == 128 ? (vkey & 3) << 2 : ((vkey >> 1) & 1) << 2)) << 4);

    int k = rg.key0(rg.i0);
    uint64_t ok = 0;
    if (tid < 2) s_odd[tid] = -1;
    __syncthreads();
    if (rg.i0 < rg.i1) ok = send(0, k);
    for (int i = rg.i0; i < rg.i1; ++i) {
        const int st = (i - rg.i0) & 1;
        const bool full = rg.full(a, k) && !~ok;
        if constexpr (!SMALL) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (!full) clean(st, i, k, ok);
        __syncthreads();  // every wave's part of tile i is there, and tile i - 1 is read
        // scores, 32 keys each
        u32x4_t kf[2][KS];
        const uint32_t ka = kbase + st * STAGE, va = vbase + st * STAGE;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < KS; ++x) kf[h][x] = lds16((ka ^ (x << 5)) + h * 64 * D);
        const int k2 = rg.key0(i + 1);
        uint64_t ok2 = 0;
        if (i + 1 < rg.i1) ok2 = send(st ^ 1, k2);
        __builtin_amdgcn_sched_barrier(0);
        // a wave at its products goes before one at its softmax (4 % of the 8192-token prompt: the
        // other has its instructions under them)
        __builtin_amdgcn_s_setprio(1);
        float16_t sc[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sc[h] = (float16_t){};
#pragma unroll
            for (int x = 0; x < KS; ++x) sc[h] = mfma32<DT>(kf[h][x], q[x], sc[h]);
        }
        // V^T operands: keys of step x, channels of tile d; the first half's latency passes
        // during the softmax
        u32x4_t vf[2][DT32];
        auto read_v = [&](int x, u32x4_t (&f)[DT32]) {
#pragma unroll
            for (int d = 0; d < DT32; ++d) {
                const uint32_t at = (va ^ (d << 6)) + x * 32 * D;
                const u32x2_t lo = tr_read(at), hi = tr_read(at + 16 * D);
                f[d] = (u32x4_t){lo.x, lo.y, hi.x, hi.y};
            }
        };
        __builtin_amdgcn_s_setprio(0);
        read_v(0, vf[0]);
        read_v(1, vf[1]);
        __builtin_amdgcn_sched_barrier(0);
        if (!full) {
            const uint64_t see = (rg.seen_bits(a, pos, k) & ok) >> (g * 4);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t half = static_cast<uint32_t>(see >> (h * 32));
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!((half >> ((e >> 2) * 8 + (e & 3))) & 1)) sc[h][e] = -INFINITY;
            }
        }
        float top = sc[0][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) top = fmaxf(top, sc[e >> 4][e & 15]);
        // (a maximum that may be 2^8 behind rescales less often, 3-5 % faster for prompts, but then
        // the largest probability, a power of two here, is rounded too: 2.2e-3 instead of 1.9e-3 of
        // an output in bf16)
        const float mn = fmaxf(m, base_of<DT>(fmaxf(top, other_half(top)) * a.scale));
        if (__any(mn > m)) {
            const float alpha = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
            sum *= alpha;
#pragma unroll
            for (int x = 0; x < DT32; ++x) acc[x] *= alpha;
            m = mn;
            far = __any(is_far(m));
        }
        if (__builtin_expect(far, 0)) {
#pragma unroll
            for (int e = 0; e < 32; ++e) sc[e >> 4][e & 15] = far_exponent(sc[e >> 4][e & 15], a.scale, m);
        }
        const float mul = far ? 1.f : a.scale;
        const float base = far || m == -INFINITY ? 0.f : m;
        u32x4_t pf[4];  // (rounded as in the few-rows kernel)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(fmaf(sc[x >> 1][(x & 1) * 8 + e], mul, -base));
                sum += p[e];
            }
            pf[x] = (u32x4_t){pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]), pack2<DT>(p[4], p[5]),
                              pack2<DT>(p[6], p[7])};
        }
        odd_seen |= s_odd[st] == i;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
#pragma unroll
            for (int d = 0; d < DT32; ++d) acc[d] = mfma32<DT>(vf[x & 1][d], pf[x], acc[d]);
            if (x < 2) read_v(x + 2, vf[x & 1]);
        }
        __builtin_amdgcn_s_setprio(0);
        k = k2;
        ok = ok2;
    }

    if (odd_seen) {
        // as in the few-rows kernel: the stages held zeros in their place
#pragma unroll 1
        for (int i = rg.i0; i < rg.i1; ++i) {
            k = rg.key0(i);
            if (rg.full(a, k) && !~__ballot(good(tab[(k + l) >> c.page_shift]))) continue;
#pragma unroll 1
            for (int key = k; key < k + 64; ++key) {
                if (!rg.any(a, key)) continue;
                const int e = tab[key >> c.page_shift];
                if (!good(e) || !rg.sees(a, pos, key)) continue;
                const uint16_t *p =
                    vb + e * c.page_stride + (key & page_mask) * c.slot_stride;
#pragma unroll
                for (int x = 0; x < DT32; ++x)
#pragma unroll
                    for (int z = 0; z < 16; ++z)
                        acc[x][z] += odd_part<DT>(p[x * 32 + (z >> 2) * 8 + g * 4 + (z & 3)]);
            }
        }
    }

    sum += other_half(sum);
    if (m == -INFINITY && sum != sum) m = 0.f;  // NaN scores only: not nothing
    if (!live) return;
    const int64_t row = static_cast<int64_t>(tok) * a.n_heads + head;
    if (a.dense == 0) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint16_t *o = a.out + row * D + g * 4;
#pragma unroll
        for (int x = 0; x < DT32; ++x)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<u32x2_t *>(o + x * 32 + e * 2) =
                    (u32x2_t){pack_out<DT>(acc[x][e] * inv, acc[x][e + 1] * inv),
                              pack_out<DT>(acc[x][e + 2] * inv, acc[x][e + 3] * inv)};
        if (a.lse && g == 0) a.lse[row] = sum == 0.f ? -INFINITY : m * kLn2 + logf(sum);
    } else {
        const int64_t at = row * a.dense + part.first + piece;
        if (m != -INFINITY) {
            float *o = a.part_o + at * D + g * 4;
#pragma unroll
            for (int x = 0; x < DT32; ++x)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    *reinterpret_cast<float4_t *>(o + x * 32 + e * 2) =
                        (float4_t){acc[x][e], acc[x][e + 1], acc[x][e + 2], acc[x][e + 3]};
        }
        if (g == 0) a.part_ml[at] = make_float2(m, sum);
    }
}

template <int DT, int D, bool SMALL>
__global__ __launch_bounds__(256, 2) void paged_attn_tile_kernel(const Cache c, const Query a,
                                                                 const Part own, const Part pre) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[kTileLds<D>];
    const int block = blockIdx.x;
    if (block < pre.groups) tile_body<DT, D, SMALL>(c, a, pre, block, lds);
    else tile_body<DT, D, SMALL>(c, a, own, block - pre.groups, lds);
}

// A prefix of many rows and few rows of each sequence in one launch, their workgroups in turn, one
// of each on a CU: the first are bound by arithmetic and latency, the second by memory.  128
// sequences behind 16384 positions 82 us, the prefix alone as long; two launches 100 us and more
// (of 8 sequences 26 us instead of 14), more and shorter pieces of the prefix 99 us: they wait for
// the other part's workgroups.
template <int DT, int D, int RB, bool SMALL>
__global__ __launch_bounds__(256, 2) void paged_attn_both_kernel(const Cache c, const Query a,
                                                                 const Few f, const Part pre) {
    constexpr int LDS = kTileLds<D> > few_lds<D>(4, RB) ? kTileLds<D> : few_lds<D>(4, RB);
    __shared__ __attribute__((aligned(16))) uint8_t lds[LDS];
    const int nf = f.groups * c.n_kv, both = 2 * (nf < pre.groups ? nf : pre.groups);
    const int i = blockIdx.x;
    if (i < both ? (i & 1) == 0 : pre.groups > nf)
        tile_body<DT, D, SMALL>(c, a, pre, i < both ? i >> 1 : i - nf, lds);
    else
        few_body<DT, D, RB, SMALL, 4>(c, a, f, i < both ? i >> 1 : i - pre.groups, lds);
}

// One workgroup per output row: O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over its
// pieces; a piece that saw nothing has m_i = -inf and no O_i.  A thread takes 4 channels of every
// kJoinThreads / (D / 4)-th piece, the threads of a channel meet in LDS in order: few rows of many
// pieces (one long sequence) are bound by the latency of their loads, which one thread a channel
// took one piece at a time (342 pieces of 28 rows: 120 us).
constexpr int kJoinThreads = 256, kJoinShift = 20;  // rows of a grid's first dimension: 2^20

template <int DT, int D, int RB>
__global__ __launch_bounds__(kJoinThreads) void paged_attn_join_kernel(const Cache c, const Query a,
                                                                       const Few f, int64_t rows) {
    constexpr int COLS = D / 4, LANES = kJoinThreads / COLS, R = 16 * RB;
    __shared__ float4_t s_o[LANES][COLS];
    __shared__ float s_m[LANES], s_l[LANES];
    const int col = threadIdx.x % COLS, lane = threadIdx.x / COLS;
    const int64_t row = blockIdx.x + (static_cast<int64_t>(blockIdx.y) << kJoinShift);
    if (row >= rows) return;
    int n[2] = {0, 0};        // pieces of few rows: of the sequence's item and of the prefix's
    int64_t slot[2] = {0, 0}; // row of the first
    if (f.groups) {
        const int tok = static_cast<int>(row / a.n_heads), head = static_cast<int>(row % a.n_heads);
        const int kvh = head / a.group;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if (x && !f.prefix) continue;
            const int2 w = f.where[(x ? c.tokens * a.group : 0) + tok * a.group + head % a.group];
            const int p = w.y >> 6, r = w.y & 63;
            // (offsets that decrease leave tokens that no item has: nothing past the slots is read)
            if (w.x < 0 || p < 1 || r >= R || w.x >= f.slots || p > f.slots - w.x) continue;
            n[x] = p;
            slot[x] = (static_cast<int64_t>(w.x) * c.n_kv + kvh) * R + r;
        }
        if (f.direct && n[0] == 1) return;  // written
    }
    const int few = n[0] + n[1], all = few + a.dense;
    float m = -INFINITY, l = 0.f;
    float4_t v = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = lane; i0 < all; i0 += 4 * LANES) {
        float2 t[4];
        float4_t o[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int i = i0 + x * LANES;
            t[x] = make_float2(-INFINITY, 0.f);
            o[x] = (float4_t){0.f, 0.f, 0.f, 0.f};
            if (i < all) {
                const int64_t at = i < n[0] ? slot[0] + static_cast<int64_t>(i) * c.n_kv * R
                                   : i < few ? slot[1] + static_cast<int64_t>(i - n[0]) * c.n_kv * R
                                             : row * a.dense + i - few;
                t[x] = (i < few ? f.part_ml : a.part_ml)[at];
                o[x] = reinterpret_cast<const float4_t *>((i < few ? f.part_o : a.part_o) + at * D)[col];
            }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if (t[x].x == -INFINITY) continue;
            const float mn = fmaxf(m, t[x].x);
            const float fo = __builtin_amdgcn_exp2f(m - mn), fn = __builtin_amdgcn_exp2f(t[x].x - mn);
            l = l * fo + t[x].y * fn;
            v = v * fo + o[x] * fn;
            m = mn;
        }
    }
    s_o[lane][col] = v;
    if (col == 0) {
        s_m[lane] = m;
        s_l[lane] = l;
    }
    __syncthreads();
    if (lane) return;
#pragma unroll
    for (int i = 0; i < LANES; ++i) m = fmaxf(m, s_m[i]);
    l = 0.f;
    v = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < LANES; ++i) {
        if (s_m[i] == -INFINITY) continue;
        const float fi = __builtin_amdgcn_exp2f(s_m[i] - m);
        l += s_l[i] * fi;
        v += s_o[i][col] * fi;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    reinterpret_cast<u32x2_t *>(a.out + row * D)[col] =
        (u32x2_t){pack_out<DT>(v[0] * inv, v[1] * inv), pack_out<DT>(v[2] * inv, v[3] * inv)};
    if (a.lse && col == 0) a.lse[row] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
}

// --------------------------------------------------------------------------------- host

int fill_cache(Cache &c, const nf4_paged_kv *kv, const int32_t *cu_q, int64_t tokens, int n_heads,
               int dtype) {
    if (!kv || (dtype != NF4_F16 && dtype != NF4_BF16)) return NF4_ERR_ARG;
    if (kv->pages < 0 || kv->page_size < 1 || kv->width < 0 || kv->batch < 0 || kv->n_kv < 1 ||
        tokens < 0 || n_heads < 1 || n_heads % kv->n_kv || kv->ld_table < kv->width)
        return NF4_ERR_ARG;
    // a position and a token times its heads stay 32-bit
    if (static_cast<int64_t>(kv->width) * kv->page_size > (1 << 30) || n_heads > 1024 ||
        tokens > (1 << 23) || tokens * n_heads > (1 << 30) || kv->batch > (1 << 20))
        return NF4_ERR_UNSUPPORTED;
    if (!cu_q && (kv->batch ? tokens % kv->batch : tokens)) return NF4_ERR_ARG;
    if (kv->head_dim != 64 && kv->head_dim != 128) return NF4_ERR_UNSUPPORTED;
    if (log2_exact(kv->page_size) < 0) return NF4_ERR_UNSUPPORTED;
    if (tokens == 0) return NF4_OK;
    if (kv->pages && kv->width && (!kv->k || !kv->v)) return NF4_ERR_ARG;
    if (kv->batch && (!kv->lens || (kv->width && !kv->table))) return NF4_ERR_ARG;
    if (kv->page_stride < 0 || kv->slot_stride < 0 || kv->head_stride < 0) return NF4_ERR_ARG;
    if (kv->slot_stride > (1 << 26)) return NF4_ERR_UNSUPPORTED;  // 15 slots in 32 bits
    if (kv->page_stride % 8 || kv->slot_stride % 8 || kv->head_stride % 8 || !aligned(kv->k, 16) ||
        !aligned(kv->v, 16) || !aligned(kv->table, 4) || !aligned(kv->lens, 4) || !aligned(cu_q, 4))
        return NF4_ERR_UNSUPPORTED;
    c.k = static_cast<uint16_t *>(kv->k);
    c.v = static_cast<uint16_t *>(kv->v);
    c.page_stride = kv->page_stride;
    c.slot_stride = kv->slot_stride;
    c.head_stride = kv->head_stride;
    c.table = kv->table;
    c.ld_table = kv->ld_table;
    c.lens = kv->lens;
    c.cu = cu_q;
    c.pages = kv->pages;
    c.page_shift = log2_exact(kv->page_size);
    // no page, or no table: no position that a key could have
    c.cap = kv->pages && kv->batch ? kv->width * kv->page_size : 0;
    c.batch = kv->batch;
    c.n_kv = kv->n_kv;
    c.tokens = static_cast<int>(tokens);
    c.uniform = kv->batch ? static_cast<int>(tokens / kv->batch) : 0;
    return NF4_OK;
}

int cut(int64_t v) { return static_cast<int>(v < (1 << 30) ? v : 1 << 30); }

int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

struct Plan {
    Few few;          // groups 0: none
    Part own, pre;    // groups 0: none
    int rb, waves;    // of the few-rows kernel
    int64_t dense, slots, where;
    size_t bytes;
};

// Sequences whose rows are few go to the kernel without LDS staging: up to 32, and up to 48 where
// equal shares count more than a third row block costs.  Those are sequences of different lengths,
// which the host does not know; what it knows is the longest (max_len, or a window), and how much
// that is over all sequences and key/value heads.  35 rows, us, this kernel and tiled:
//   longest 16000, 64 sequences of 40 to it, 4 heads of 128    227  287   6 of 64  228  364
//   longest 16000, 8 sequences, 4 heads 37  41, 16 of one head 31  29, 24 of one head 37  40
//   longest 9000, 16 sequences, 4 heads 49  54, 8 sequences    31  29
//   5000 and 6000, 8 and 16 sequences,  4 heads 30  24, 43  40; 64 of 4300 each 121 118
//   one sequence of 9000  20  19; in windows of 1024 58  44; a prefix of 2001 22  15
// Where all it knows is the table's width, tiles would be cut for that, and equal shares are for
// what is there (4 heads, 16 sequences of 40 to 2000 in tables of 8192 23  46, of 5120 23  34; 64
// of 5000 in 5120 129  135; against it 64 of 40 to 2000 of 8 heads 96  72, and one of 500 19  13).
// Its launch is a workgroup on every CU (kFewSlots): 64 KB in flight on each are enough for the
// memory's rate, and more workgroups mean shorter shares and more pieces (131071 keys, 64 ragged
// sequences: 512 workgroups 63.5 and 215 us, 256 60.6 and 212.7).  Where no sequence is longer than
// kWholeKeys and all of them fit the card, a workgroup of 8 waves takes a whole sequence, and there
// is nothing to join.  Tiled parts are cut until the launch has kTileSlots workgroups.
constexpr int kFewRows = 32, kFewRowsLong = 48, kLongKeys = 8192, kLongWidth = 4096, kFewSlots = 256,
              kTileSlots = 512, kWholeKeys = 1024;
constexpr int64_t kLongWork = 3 << 17;  // keys of all sequences and heads

// `rows` > 0: cutting the part is what makes a join of that many rows necessary.  A tile takes
// 2 us, a join 4 us and 0.15 ns for each row and each of its pieces (written and read): 6 chunks of
// 143 to 431 tokens in windows of 210 go from 34 us in 3 pieces to 18 in one, 2 chunks of 21 to 65
// tokens behind 1500 stay at 16 us in 25 (20 in 6).
Part tile_part(bool prefix, int64_t rows, int64_t blocks, int n_kv, int64_t keys, int slots) {
    Part p{};
    const int tiles = ceil_div(keys, 64) + 1;
    const int64_t groups = blocks * n_kv;
    int64_t most = slots / (groups ? groups : 1), splits = 1;
    most = most < 1 ? 1 : most > tiles ? tiles : most;
    double best = 2.0 * tiles;
    for (int64_t n = most; n > 1; n /= 2) {
        const double t = 2.0 * ceil_div(tiles, n) + (rows ? 4.0 + 1.5e-4 * rows * (n + 2) : 0.0);
        if (t < best) {
            best = t;
            splits = n;
        }
    }
    p.prefix = prefix ? 1 : 0;
    p.min_tiles = ceil_div(tiles, splits);
    p.splits = ceil_div(tiles, p.min_tiles);
    p.blocks = static_cast<int>(blocks);
    p.groups = cut(groups * p.splits);
    return p;
}

Plan make_plan(const Cache &c, int n_heads, int window, int sinks, int shared, int64_t max_q,
               int64_t max_len, int head_dim) {
    const int64_t group = n_heads / c.n_kv, all_rows = c.tokens * group;
    int64_t longest = c.cu ? (max_q && max_q < c.tokens ? max_q : c.tokens) : c.uniform;
    const int64_t len = max_len && max_len < c.cap ? max_len : c.cap;
    int64_t span = len > shared ? len - shared : 0;
    if (window && span > static_cast<int64_t>(window) + longest + sinks) span = window + longest + sinks;
    const int64_t pre_keys = len < shared ? len : shared;
    const int seqs = c.batch + (c.cu ? 1 : 0);  // with offsets: and the tokens past the last
    const bool few_pre = shared && all_rows <= kFewRows;
    const bool told = max_len || span < c.cap;
    const bool uneven = !shared && (told ? span > kLongKeys && span * c.batch * c.n_kv >= kLongWork
                                         : span > kLongWidth && c.batch > 1);
    const bool few_own = longest * group <= (uneven ? kFewRowsLong : kFewRows);
    Plan p{};
    if (few_own) {
        Few &f = p.few;
        const int64_t rows = few_pre ? all_rows : longest * group;
        p.rb = rows <= 16 ? 1 : rows <= 32 ? 2 : 3;
        f.seqs = seqs;
        f.prefix = few_pre ? 1 : 0;
        f.direct = shared ? 0 : 1;
        f.items = static_cast<int>(all_rows / (16 * p.rb)) + seqs +
                  (few_pre ? ceil_div(all_rows, 16 * p.rb) : 0);
        f.whole = !shared && p.rb == 1 && span <= kWholeKeys &&
                  static_cast<int64_t>(f.items) * c.n_kv <= 2 * 256;
        p.waves = f.whole ? 8 : 4;
        f.min_units = 2;
        int64_t units = f.items * (span / (32 * p.waves) + 2) + pre_keys / 128 + 2;
        // (three row blocks: one workgroup's registers and LDS are a CU's, one past the CUs would
        // start when the others end: 258 of 6 heads 493 us where 252 are 316)
        int64_t groups = p.rb < 3 ? ceil_div(kFewSlots, c.n_kv) : c.n_kv < kFewSlots ? kFewSlots / c.n_kv : 1;
        groups = groups < units / f.min_units ? groups : units / f.min_units;
        f.groups = f.whole ? (c.cu ? f.items : seqs) : static_cast<int>(groups < 1 ? 1 : groups);
        if (!f.whole) {
            p.slots = f.slots = f.groups + f.items;
            p.where = all_rows * (1 + f.prefix);
        }
    } else {
        const int64_t blocks = c.cu ? all_rows / kRows + seqs
                                    : static_cast<int64_t>(c.batch) * ceil_div(longest * group, kRows);
        // (a row block's window, not all of a sequence's)
        const int64_t seen = static_cast<int64_t>(window) + kRows / group + 1 + sinks;
        p.own = tile_part(false, shared ? 0 : static_cast<int64_t>(c.tokens) * n_heads, blocks, c.n_kv, window && seen < span ? seen : span, kTileSlots);
    }
    if (shared && !few_pre)
        p.pre = tile_part(true, 0, ceil_div(all_rows, kRows), c.n_kv, pre_keys,
                          few_own ? kTileSlots / 2 : kTileSlots);
    p.own.first = p.pre.groups ? p.pre.splits : 0;
    p.dense = p.own.first + (p.own.groups ? p.own.splits : 0);
    if (!shared && p.dense == 1) p.dense = 0;
    p.bytes = (p.dense * c.tokens * n_heads + p.slots * c.n_kv * 16 * p.rb) * (4 * head_dim + 8) +
              p.where * 8;
    return p;
}

template <int DT, int D, bool SMALL>
int launch(const Cache &c, const Query &a, const Plan &p, hipStream_t s) {
    const int64_t nf = static_cast<int64_t>(p.few.groups) * c.n_kv;
    const int64_t groups = nf + p.pre.groups + p.own.groups;
    if (groups == 0) return NF4_OK;
    if (groups > (1 << 23)) return NF4_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(groups));
#define NF4_FEW(RB, W)                                                                              \
    hipLaunchKernelGGL((paged_attn_few_kernel<DT, D, RB, SMALL, W>), grid, dim3(64 * W), 0, s, c, a, \
                       p.few)
#define NF4_BOTH(RB)                                                                                \
    hipLaunchKernelGGL((paged_attn_both_kernel<DT, D, RB, SMALL>), grid, dim3(256), 0, s, c, a,      \
                       p.few, p.pre)
    if (nf == 0)
        hipLaunchKernelGGL((paged_attn_tile_kernel<DT, D, SMALL>), grid, dim3(256), 0, s, c, a, p.own,
                           p.pre);
    else if (p.pre.groups)
        if (p.rb == 1) NF4_BOTH(1);
        else NF4_BOTH(2);
    else if (p.few.whole) NF4_FEW(1, 8);
    else if (p.rb == 1) NF4_FEW(1, 4);
    else if (p.rb == 2) NF4_FEW(2, 4);
    else NF4_FEW(3, 4);
#undef NF4_FEW
#undef NF4_BOTH
    const int st = status_of(hipGetLastError());
    if (st != NF4_OK || p.bytes == 0) return st;
    const int64_t rows = static_cast<int64_t>(c.tokens) * a.n_heads;
    const dim3 joins(static_cast<unsigned>(rows < (1 << kJoinShift) ? rows : 1 << kJoinShift),
                     static_cast<unsigned>((rows + (1 << kJoinShift) - 1) >> kJoinShift));
#define NF4_JOIN(RB)                                                                                \
    hipLaunchKernelGGL((paged_attn_join_kernel<DT, D, RB>), joins, dim3(kJoinThreads), 0, s, c, a,   \
                       p.few, rows)
    if (p.rb == 3) NF4_JOIN(3);
    else if (p.rb == 2) NF4_JOIN(2);
    else NF4_JOIN(1);
#undef NF4_JOIN
    return status_of(hipGetLastError());
}

template <int DT>
int launch_of(const Cache &c, const Query &a, const Plan &p, int head_dim, hipStream_t s) {
    // per-lane page addresses: for pages under 16 slots, and for pages that span 2^31 bytes
    const bool small = c.page_shift < 4 || c.slot_stride * 2 << c.page_shift >= 0x7fffffff;
    if (head_dim == 128)
        return small ? launch<DT, 128, true>(c, a, p, s) : launch<DT, 128, false>(c, a, p, s);
    return small ? launch<DT, 64, true>(c, a, p, s) : launch<DT, 64, false>(c, a, p, s);
}

}  // namespace

extern "C" int nf4_paged_append(const nf4_paged_kv *kv, const void *qkv, int64_t ld_qkv,
                                const float *cos_t, const float *sin_t, int64_t rope_rows,
                                const int32_t *cu_q, void *q, int64_t tokens, int n_heads,
                                int dtype, void *stream) {
    Cache c{};
    const int st = fill_cache(c, kv, cu_q, tokens, n_heads, dtype);
    if (st != NF4_OK) return st;
    if (rope_rows < 0 || ld_qkv < static_cast<int64_t>(n_heads + 2 * kv->n_kv) * kv->head_dim)
        return NF4_ERR_ARG;
    if (tokens == 0) return NF4_OK;
    if (!qkv || !q || (rope_rows && (!cos_t || !sin_t))) return NF4_ERR_ARG;
    if (ld_qkv % 8 || !aligned(qkv, 16) || !aligned(q, 16) || !aligned(cos_t, 16) ||
        !aligned(sin_t, 16))
        return NF4_ERR_UNSUPPORTED;
    const int rows = rope_rows > 0x7fffffff ? 0x7fffffff : static_cast<int>(rope_rows);
    auto s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(tokens));
    auto X = static_cast<const uint16_t *>(qkv);
    auto Q = static_cast<uint16_t *>(q);
    if (dtype == NF4_BF16)
        hipLaunchKernelGGL(paged_append_kernel<NF4_BF16>, grid, dim3(kAppendThreads), 0, s, c, X,
                           ld_qkv, cos_t, sin_t, rows, Q, n_heads, kv->head_dim);
    else
        hipLaunchKernelGGL(paged_append_kernel<NF4_F16>, grid, dim3(kAppendThreads), 0, s, c, X,
                           ld_qkv, cos_t, sin_t, rows, Q, n_heads, kv->head_dim);
    return status_of(hipGetLastError());
}

extern "C" size_t nf4_paged_attn_workspace(const nf4_paged_kv *kv, const int32_t *cu_q,
                                           int64_t tokens, int n_heads, int64_t window,
                                           int64_t sinks, int64_t shared, int64_t max_q,
                                           int64_t max_len) {
    Cache c{};
    if (fill_cache(c, kv, cu_q, tokens, n_heads, NF4_F16) != NF4_OK || tokens == 0) return 0;
    if (window < 0 || sinks < 0 || shared < 0 || max_q < 0 || max_len < 0) return 0;
    return make_plan(c, n_heads, cut(window), cut(sinks), cut(shared), max_q, max_len,
                     kv->head_dim).bytes;
}

extern "C" int nf4_paged_attn(const nf4_paged_kv *kv, const void *q, int64_t ld_tok,
                              int64_t ld_head, const int32_t *cu_q, void *out, float *lse,
                              int64_t tokens, int n_heads, float scale, int64_t window,
                              int64_t sinks, int64_t shared, int64_t max_q, int64_t max_len,
                              int dtype, void *workspace, size_t workspace_bytes, void *stream) {
    Cache c{};
    const int st = fill_cache(c, kv, cu_q, tokens, n_heads, dtype);
    if (st != NF4_OK) return st;
    if (window < 0 || sinks < 0 || shared < 0 || max_q < 0 || max_len < 0) return NF4_ERR_ARG;
    const float scale2 = fabsf(scale) * kLog2e;
    if (!(scale2 < INFINITY)) return NF4_ERR_ARG;  // NaN too
    if (tokens == 0) return NF4_OK;
    if (!q || !out) return NF4_ERR_ARG;
    if (ld_tok < 0 || ld_head < 0) return NF4_ERR_ARG;
    if (ld_tok % 8 || ld_head % 8 || !aligned(q, 16) || !aligned(out, 16) || !aligned(lse, 4))
        return NF4_ERR_UNSUPPORTED;
    Query a{};
    a.q = static_cast<const uint16_t *>(q);
    a.ld_tok = ld_tok;
    a.ld_head = ld_head;
    a.out = static_cast<uint16_t *>(out);
    a.lse = lse;
    a.n_heads = n_heads;
    a.group = n_heads / c.n_kv;
    a.window = cut(window);
    a.sinks = cut(sinks);
    a.shared = cut(shared);
    a.flip = scale < 0.f ? 0x80008000u : 0u;
    a.scale = fmaxf(scale2, 1.2e-38f);  // not 0 (a hidden score is -inf): a normal number's least
    Plan p = make_plan(c, n_heads, a.window, a.sinks, a.shared, max_q, max_len, kv->head_dim);
    a.dense = p.dense;
    if (p.bytes) {
        if (!workspace || workspace_bytes < p.bytes) return NF4_ERR_WORKSPACE;
        if (!aligned(workspace, 16)) return NF4_ERR_UNSUPPORTED;
        const int64_t rows = p.dense * tokens * n_heads, few = p.slots * c.n_kv * 16 * p.rb;
        a.part_o = static_cast<float *>(workspace);
        p.few.part_o = a.part_o + rows * kv->head_dim;
        a.part_ml = reinterpret_cast<float2 *>(p.few.part_o + few * kv->head_dim);
        p.few.part_ml = a.part_ml + rows;
        p.few.where = reinterpret_cast<int2 *>(p.few.part_ml + few);
    }
    auto s = static_cast<hipStream_t>(stream);
    return dtype == NF4_BF16 ? launch_of<NF4_BF16>(c, a, p, kv->head_dim, s)
                             : launch_of<NF4_F16>(c, a, p, kv->head_dim, s);
}
