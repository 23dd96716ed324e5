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
// once; v heads are copied the same way.
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
// Parts.  A launch covers the positions [shared, end) of each sequence through its own table
// row, or (prefix) [0, shared) through row 0 for the rows of the whole batch.  The tiles that
// some row of a workgroup sees (sink tiles, then window tiles) are cut into `splits` pieces; with
// one piece in all the workgroup writes the output, else (maximum, sum, unscaled output) in fp32
// for paged_attn_join_kernel.

struct Query {
    const uint16_t *q;
    int64_t ld_tok, ld_head;
    uint16_t *out;
    float *lse;
    float *part_o;   // [tokens * n_heads][pieces][D]
    float2 *part_ml; // [tokens * n_heads][pieces]
    int pieces;      // of all the parts
    int n_heads, group, window, sinks, shared;
    float scale;     // of the scores in units of log 2, positive
    uint32_t flip;   // sign bits of a query pair, where the scale is negative
};

struct Part {
    int prefix;     // 1: positions below `shared`, the whole batch's rows
    int splits;     // pieces of this part
    int first;      // index of its first piece
    int min_tiles;  // tiles of a piece, at least
    int blocks;     // row blocks (tiled kernel)
};

constexpr int kNowhere = -(1 << 30);  // the position of a row that is not there

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

// What a workgroup's rows (positions pmin .. pmax) see of a part: keys of [lo, hi) that are at
// most at the row's position, and past its window's start or below `sinks`; tiles of 2^SH keys,
// first those of the sinks, then those of the windows.
template <int SH>
struct Range {
    int lo, hi, pmin, pmax;
    int sink0, sinks_n, win0, n;  // tiles
    int i0, i1;                   // of this piece

    __device__ __forceinline__ void set(const Cache &c, const Query &a, const Part &part, int piece) {
        const int end = pmax + 1 < c.cap ? pmax + 1 : c.cap;
        lo = part.prefix ? 0 : a.shared;
        hi = part.prefix && a.shared < end ? a.shared : end;
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
        int per = (n + part.splits - 1) / part.splits;
        per = per > part.min_tiles ? per : part.min_tiles;
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

// 8 consecutive values of a query row, its sign as the scale's.
__device__ __forceinline__ u32x4_t load_q(const Query &a, int tok, int head, int d) {
    u32x4_t r = *reinterpret_cast<const u32x4_t *>(a.q + tok * a.ld_tok + head * a.ld_head + d);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] ^= a.flip;
    return r;
}

// ------------------------------------------------------------- few rows (decoding)
//
// At most 16 RB rows (more are taken in turns): the bytes of the cache are all that counts, and
// no key is used often enough for LDS to pay.  Each of a workgroup's 4 waves takes every fourth
// 32-key slab on its own, straight from memory into MFMA operands: a lane loads 16 bytes of a key
// (rows of K are A-operand rows as they lie) and 16 bytes (8 channels) of 8 of its V rows, and
// turns the 8x8 block of V into operands by byte permutes, which is free beside the memory
// (channel e of each lane's 8 forms one product, so the order of channels is a permuted one).
// The next slab's keys are loaded as soon as the scores are formed and its values as soon as they
// are used, so that a wave always has loads in flight; the 4 waves' results meet in LDS.

template <int DT, int D, int RB, bool SMALL>
__global__ __launch_bounds__(256, RB == 1 ? 3 : 2) void paged_attn_few_kernel(const Cache c, const Query a,
                                                             const Part part) {
    constexpr int KC = D / 32, VE = D / 16, LD = D + 4;  // K chunks, V values a lane, LDS row
    __shared__ float s_o[4][16 * RB][LD];
    __shared__ float s_ml[4][16 * RB][2];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
    const int g = l >> 4, n = l & 15;
    const int kvh = blockIdx.x % c.n_kv, y = blockIdx.x / c.n_kv;
    const int piece = y % part.splits, item = y / part.splits;
    const int b = part.prefix ? 0 : item;
    Seq s = {0, c.tokens, 0};
    if (!part.prefix) s = seq_at(c, b);
    const int rows = s.n * a.group;
    const int32_t *tab = c.table + b * c.ld_table;
    const char *kb = reinterpret_cast<const char *>(c.k + kvh * c.head_stride);
    const char *vb = reinterpret_cast<const char *>(c.v + kvh * c.head_stride);
    const uint32_t stride2 = static_cast<uint32_t>(c.slot_stride) * 2;
    const int page_mask = (1 << c.page_shift) - 1;

    for (int r0 = part.prefix ? item * 16 * RB : 0; r0 < rows; r0 += 16 * RB) {
        // this lane's rows and their positions
        u32x4_t q[RB][KC];
        int pos[RB], pmin = 0x7fffffff, pmax = kNowhere;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = r0 + rb * 16 + n;
            pos[rb] = kNowhere;
#pragma unroll
            for (int k = 0; k < KC; ++k) q[rb][k] = (u32x4_t){0, 0, 0, 0};
            if (r < rows) {
                const int tok = s.q0 + r / a.group, head = kvh * a.group + r % a.group;
                pos[rb] = part.prefix ? position_of(c, tok) : s.p0 + r / a.group;
                pmin = pos[rb] < pmin ? pos[rb] : pmin;
                pmax = pos[rb] > pmax ? pos[rb] : pmax;
#pragma unroll
                for (int k = 0; k < KC; ++k) q[rb][k] = load_q(a, tok, head, k * 32 + g * 8);
            }
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const int x = __shfl_xor(pmin, o), z = __shfl_xor(pmax, o);
            pmin = x < pmin ? x : pmin;
            pmax = z > pmax ? z : pmax;
        }
        Range<5> rg;
        rg.pmin = __builtin_amdgcn_readfirstlane(pmin);
        rg.pmax = __builtin_amdgcn_readfirstlane(pmax);
        rg.set(c, a, part, piece);

        float m[RB], sum[RB];
        float4_t acc[RB][VE];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            m[rb] = -INFINITY;
            sum[rb] = 0.f;
#pragma unroll
            for (int e = 0; e < VE; ++e) acc[rb][e] = (float4_t){0.f, 0.f, 0.f, 0.f};
        }

        // page entries of the slab at key k: of its two 16-key halves, or (pages under 16) of
        // key k + l % 32
        auto entry = [&](int k, int half) {
            if constexpr (SMALL) {
                const int j = k + (l & 31);
                return j < c.cap ? tab[j >> c.page_shift] : -1;
            } else {
                return k + half * 16 < c.cap ? sload(tab + ((k + half * 16) >> c.page_shift)) : -1;
            }
        };
        auto good = [&](int e) { return static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages); };
        // key i (0 .. 31) of the slab, in bytes of k or v: where there is no page, page 0's
        auto slot = [&](int e0, int e1, int k, int i) -> int64_t {
            int e;
            if constexpr (SMALL) e = __shfl(e0, i);
            else e = i < 16 ? e0 : e1;
            e = good(e) ? e : 0;
            return (e * c.page_stride + ((k + i) & page_mask) * c.slot_stride) * 2;
        };
        u32x4_t kr[2][KC];
        u32x4_t vr[8];
        // a half slab's page and first slot are the wave's (a scalar base), the rest the lane's
        auto load_k = [&](int e0, int e1, int k) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char *p = SMALL ? kb + slot(e0, e1, k, h * 16 + n) : kb + slot(e0, e1, k, h * 16);
                const uint32_t o = SMALL ? g * 16 : n * stride2 + g * 16;
#pragma unroll
                for (int x = 0; x < KC; ++x)
                    kr[h][x] = *reinterpret_cast<const u32x4_t *>(p + (o + x * 64));
            }
        };
        auto load_v = [&](int e0, int e1, int k) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int h = j >> 2, i = g * 4 + (j & 3);
                const char *p = SMALL ? vb + slot(e0, e1, k, h * 16 + i) : vb + slot(e0, e1, k, h * 16);
                const uint32_t o = SMALL ? n * VE * 2 : i * stride2 + n * VE * 2;
                if constexpr (D == 128) {
                    vr[j] = *reinterpret_cast<const u32x4_t *>(p + o);
                } else {
                    const u32x2_t t = *reinterpret_cast<const u32x2_t *>(p + o);
                    vr[j] = (u32x4_t){t.x, t.y, 0, 0};
                }
            }
        };

        int i = rg.i0 + w, k = rg.key0(i), e0 = -1, e1 = -1, f0 = -1, f1 = -1;
        if (i < rg.i1) {
            e0 = entry(k, 0);
            e1 = entry(k, 1);
            load_k(e0, e1, k);
            load_v(e0, e1, k);
        }
        int k2 = rg.key0(i + 4);
        if (i + 4 < rg.i1) {
            f0 = entry(k2, 0);
            f1 = entry(k2, 1);
        }
        while (i < rg.i1) {
            const bool more = i + 4 < rg.i1;
            float4_t st[RB][2];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    st[rb][h] = (float4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int x = 0; x < KC; ++x) st[rb][h] = mfma16<DT>(kr[h][x], q[rb][x], st[rb][h]);
                }
            uint32_t ok;  // keys whose page is there
            if constexpr (SMALL) ok = static_cast<uint32_t>(__ballot(good(e0)));
            else ok = (good(e0) ? 0xffffu : 0u) | (good(e1) ? 0xffff0000u : 0u);
            if (more) load_k(f0, f1, k2);
            const bool full = rg.full(a, k) && ok == 0xffffffffu;
            bool odd = false;  // an infinity or NaN among values that not every row sees
            if (!full) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = (j >> 2) * 16 + g * 4 + (j & 3);
                    if (!((ok >> key) & 1) || !rg.any(a, k + key)) vr[j] = (u32x4_t){0, 0, 0, 0};
#pragma unroll
                    for (int x = 0; x < VE / 2; ++x) odd |= not_finite<DT>(vr[j][x]);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb)
                        if (!((ok >> key) & 1) || !rg.sees(a, pos[rb], k + key))
                            st[rb][j >> 2][j & 3] = -INFINITY;
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
                const float mn = fmaxf(m[rb], top * a.scale);
                if (__any(mn > m[rb])) {
                    const float alpha = mn > m[rb] ? __builtin_amdgcn_exp2f(m[rb] - mn) : 1.f;
                    sum[rb] *= alpha;
#pragma unroll
                    for (int e = 0; e < VE; ++e) acc[rb][e] *= alpha;
                    m[rb] = mn;
                }
                const float base = m[rb] == -INFINITY ? 0.f : m[rb];
                float p[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    p[j] = __builtin_amdgcn_exp2f(fmaf(st[rb][j >> 2][j & 3], a.scale, -base));
                    sum[rb] += p[j];
                }
                // probabilities in the 16-bit type for the MFMA; their sum stays unrounded
                pf[rb] = (u32x4_t){pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]),
                                   pack2<DT>(p[4], p[5]), pack2<DT>(p[6], p[7])};
            }
            if (__any(odd)) {
                // 0 times such a value is no 0: they are added to the rows that see them (a
                // probability above 0 leaves an infinity or NaN what it is) and leave the products
#pragma unroll 1
                for (int key = 0; key < 32; ++key) {
                    if (!((ok >> key) & 1) || !rg.any(a, k + key)) continue;
                    const char *p = vb + (tab[(k + key) >> c.page_shift] * c.page_stride +
                                          ((k + key) & page_mask) * c.slot_stride) * 2;
                    bool see[RB];
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) see[rb] = rg.sees(a, pos[rb], k + key);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const u32x2_t *vp = reinterpret_cast<const u32x2_t *>(p + (g * 4 + x) * VE * 2);
#pragma unroll
                        for (int e = 0; e < VE; e += 4) {
                            const u32x2_t t = vp[e / 4];
#pragma unroll
                            for (int z = 0; z < 4; ++z) {
                                const float o = odd_part<DT>(z & 1 ? t[z >> 1] >> 16 : t[z >> 1]);
#pragma unroll
                                for (int rb = 0; rb < RB; ++rb) acc[rb][e + z][x] += see[rb] ? o : 0.f;
                            }
                        }
                    }
                }
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
            if (more) {
                load_v(f0, f1, k2);
                e0 = f0;
                e1 = f1;
                const int k3 = rg.key0(i + 8);
                if (i + 8 < rg.i1) {
                    f0 = entry(k3, 0);
                    f1 = entry(k3, 1);
                }
                k = k2;
                k2 = k3;
            }
            i += 4;
        }

        // the 4 waves' parts: each scaled to the common maximum, summed over LDS in wave order
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            sum[rb] += __shfl_xor(sum[rb], 16);
            sum[rb] += __shfl_xor(sum[rb], 32);
            if (g == 0) {
                s_ml[w][rb * 16 + n][0] = m[rb];
                s_ml[w][rb * 16 + n][1] = sum[rb];
            }
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int e = 0; e < VE; e += 4)
                    *reinterpret_cast<float4_t *>(&s_o[w][rb * 16 + n][(g * 4 + x) * VE + e]) =
                        (float4_t){acc[rb][e][x], acc[rb][e + 1][x], acc[rb][e + 2][x], acc[rb][e + 3][x]};
        }
        __syncthreads();
        for (int u = threadIdx.x; u < 16 * RB * (D / 8); u += 256) {
            const int r = u / (D / 8), d = (u % (D / 8)) * 8;
            if (r0 + r >= rows) continue;
            float mm = -INFINITY, ll = 0.f, o[8] = {};
#pragma unroll
            for (int x = 0; x < 4; ++x) mm = fmaxf(mm, s_ml[x][r][0]);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float mw = s_ml[x][r][0], f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - mm);
                ll += s_ml[x][r][1] * f;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] += s_o[x][r][d + e] * f;
            }
            const int64_t row = static_cast<int64_t>(s.q0 + (r0 + r) / a.group) * a.n_heads +
                                kvh * a.group + (r0 + r) % a.group;
            if (a.pieces == 1) {
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] *= inv;
                *reinterpret_cast<u32x4_t *>(a.out + row * D + d) = pack8<DT>(o);
                if (a.lse && d == 0) a.lse[row] = ll == 0.f ? -INFINITY : mm * kLn2 + logf(ll);
            } else {
                const int64_t at = row * a.pieces + part.first + piece;
                if (mm != -INFINITY) {
                    float4_t *po = reinterpret_cast<float4_t *>(a.part_o + at * D + d);
                    po[0] = (float4_t){o[0], o[1], o[2], o[3]};
                    po[1] = (float4_t){o[4], o[5], o[6], o[7]};
                }
                if (d == 0) a.part_ml[at] = make_float2(mm, ll);
            }
        }
        if (part.prefix) return;  // the other rows are other workgroups'
        __syncthreads();
    }
}

// ------------------------------------------------------------------ many rows (prompts)
//
// 128 rows a workgroup, 32 a wave on v_mfma_f32_32x32x16, over 64-key tiles: K and V tiles go
// through LDS, loaded into registers while the tile before is used (two LDS stages, one barrier
// a tile).  16-byte chunk ch of K's row r lies at chunk ch ^ (r & 15) (128 channels; 64: ch ^
// (r / 2 & 7)): the 16 lanes that LDS serves at a time then read 16 rows from 16 different bank
// groups.  V is read transposed (ds_read_b64_tr_b16: 4 keys of a channel a lane) from rows whose
// 64-byte blocks are exchanged by the key's low bits, 4 keys x 64 bytes on all banks.

typedef short v4i16_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16_t lds_v4i16_t;

__device__ __forceinline__ u32x2_t tr_read(const uint8_t *s, int off) {
    return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_v4i16_t *)((__attribute__((address_space(3))) uint8_t *)s + off)));
}

constexpr int kRows = 128;

template <int DT, int D, bool SMALL>
__global__ __launch_bounds__(256, 2) void paged_attn_tile_kernel(const Cache c, const Query a,
                                                                 const Part part) {
    constexpr int CH = D / 8, KS = D / 16, DT32 = D / 32;  // 16-byte chunks of a row, k steps, d tiles
    constexpr int RPP = 256 / CH, PASS = 64 / RPP;         // rows a pass of the workgroup loads
    __shared__ __attribute__((aligned(16))) uint8_t s_k[2][64 * D * 2];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[2][64 * D * 2];
    __shared__ int s_odd[2];  // the stage's tile, where its values hold an infinity or NaN
    __shared__ int s_p[8];
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63;
    const int g = l >> 5, n = l & 31;
    const int kvh = blockIdx.x % c.n_kv, y = blockIdx.x / c.n_kv;
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
        s = seq_at(c, b);
    }
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
    rg.set(c, a, part, piece);

    float m = -INFINITY, sum = 0.f;
    float16_t acc[DT32];
#pragma unroll
    for (int x = 0; x < DT32; ++x) acc[x] = (float16_t){};

    // ---- staging: thread's row of a pass and its chunk
    const int srow = tid / CH, sch = tid % CH;
    auto k_at = [&](int row, int ch) {  // byte of a K chunk in its stage
        return row * D * 2 + ((ch ^ (D == 128 ? (row & 15) : ((row >> 1) & 7))) << 4);
    };
    auto v_at = [&](int row, int ch) {
        return row * D * 2 + ((ch ^ (D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2)) << 4);
    };
    auto good = [&](int e) { return static_cast<uint32_t>(e) < static_cast<uint32_t>(c.pages); };
    // page entries of the tile at key k: of its 16-key quarters, or (pages under 16) key k + l's
    struct Entries { int e[4]; };
    auto entries = [&](int k) {
        Entries t;
        if constexpr (SMALL) {
            t.e[0] = k + l < c.cap ? tab[(k + l) >> c.page_shift] : -1;
        } else {
#pragma unroll
            for (int x = 0; x < 4; ++x)
                t.e[x] = k + 16 * x < c.cap ? sload(tab + ((k + 16 * x) >> c.page_shift)) : -1;
        }
        return t;
    };
    auto there = [&](const Entries &t) -> uint64_t {  // keys whose page is there
        if constexpr (SMALL) {
            return __ballot(good(t.e[0]));
        } else {
            uint64_t v = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) v |= good(t.e[x]) ? 0xffffull << (16 * x) : 0;
            return v;
        }
    };
    u32x4_t kst[PASS], vst[PASS];
    auto load = [&](const Entries &t, int k) {
#pragma unroll
        for (int x = 0; x < PASS; ++x) {
            const int row = x * RPP + srow;
            int e;
            if constexpr (SMALL) e = __shfl(t.e[0], row);
            else if constexpr (D == 128) e = t.e[x];
            else e = w < 2 ? t.e[2 * x] : t.e[2 * x + 1];
            e = good(e) ? e : 0;
            const int64_t at = e * c.page_stride + kvh * c.head_stride +
                               ((k + row) & page_mask) * c.slot_stride + sch * 8;
            kst[x] = *reinterpret_cast<const u32x4_t *>(c.k + at);
            vst[x] = *reinterpret_cast<const u32x4_t *>(c.v + at);
        }
    };
    auto store = [&](int st, int i, int k, uint64_t ok) {
        if (!rg.full(a, k) || ~ok) {
            bool odd = false;
#pragma unroll
            for (int x = 0; x < PASS; ++x) {
                const int row = x * RPP + srow;
                if (!((ok >> row) & 1) || !rg.any(a, k + row)) vst[x] = (u32x4_t){0, 0, 0, 0};
#pragma unroll
                for (int z = 0; z < 4; ++z) odd |= not_finite<DT>(vst[x][z]);
            }
            if (odd) {
#pragma unroll
                for (int x = 0; x < PASS; ++x)
#pragma unroll
                    for (int z = 0; z < 4; ++z) vst[x][z] = finite_or_zero<DT>(vst[x][z]);
                s_odd[st] = i;
            }
        }
#pragma unroll
        for (int x = 0; x < PASS; ++x) {
            const int row = x * RPP + srow;
            *reinterpret_cast<u32x4_t *>(s_k[st] + k_at(row, sch)) = kst[x];
            *reinterpret_cast<u32x4_t *>(s_v[st] + v_at(row, sch)) = vst[x];
        }
    };

    // ---- operand addresses of this lane
    const int krow = n * D * 2, kx = D == 128 ? (n & 15) : ((n >> 1) & 7);
    const int vkey = g * 4 + ((l & 15) >> 2);  // key (of 16) and chunk that it points at
    const int vch = ((l >> 4) & 1) * 2 + ((l & 3) >> 1);
    const int vbase = vkey * D * 2 + (l & 1) * 8;
    const int vx = D == 128 ? (vkey & 3) << 2 : ((vkey >> 1) & 1) << 2;

    Entries cur{}, nxt{};
    int k = 0, k2 = 0;
    uint64_t ok = 0;
    if (tid < 2) s_odd[tid] = -1;
    __syncthreads();
    if (rg.i0 < rg.i1) {
        k = rg.key0(rg.i0);
        cur = entries(k);
        load(cur, k);
        ok = there(cur);
        store(0, rg.i0, k, ok);
        k2 = rg.key0(rg.i0 + 1);
        if (rg.i0 + 1 < rg.i1) nxt = entries(k2);
    }
    __syncthreads();
    for (int i = rg.i0; i < rg.i1; ++i) {
        const int st = (i - rg.i0) & 1;
        const bool more = i + 1 < rg.i1;
        if (more) load(nxt, k2);
        Entries nxt2{};
        const int k3 = rg.key0(i + 2);
        if (i + 2 < rg.i1) nxt2 = entries(k3);
        // scores, 32 keys each
        float16_t sc[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sc[h] = (float16_t){};
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                const u32x4_t f = *reinterpret_cast<const u32x4_t *>(
                    s_k[st] + h * 32 * D * 2 + krow + (((2 * x + g) ^ kx) << 4));
                sc[h] = mfma32<DT>(f, q[x], sc[h]);
            }
        }
        const bool full = rg.full(a, k) && !~ok;
        if (!full) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int key = h * 32 + (e >> 2) * 8 + g * 4 + (e & 3);
                    if (!((ok >> key) & 1) || !rg.sees(a, pos, k + key)) sc[h][e] = -INFINITY;
                }
        }
        float top = sc[0][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) top = fmaxf(top, sc[e >> 4][e & 15]);
        top = fmaxf(top, __shfl_xor(top, 32)) * a.scale;
        if (__any(top > m)) {
            const float mn = fmaxf(m, top), alpha = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
            sum *= alpha;
#pragma unroll
            for (int x = 0; x < DT32; ++x) acc[x] *= alpha;
            m = mn;
        }
        const float base = m == -INFINITY ? 0.f : m;
        u32x4_t pf[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(fmaf(sc[x >> 1][(x & 1) * 8 + e], a.scale, -base));
                sum += p[e];
            }
            pf[x] = (u32x4_t){pack2<DT>(p[0], p[1]), pack2<DT>(p[2], p[3]), pack2<DT>(p[4], p[5]),
                              pack2<DT>(p[6], p[7])};
        }
        if (s_odd[st] == i) {
            // as in the few-rows kernel: the stage holds zeros in their place
#pragma unroll 1
            for (int key = 0; key < 64; ++key) {
                if (!((ok >> key) & 1) || !rg.any(a, k + key)) continue;
                const uint16_t *p = c.v + tab[(k + key) >> c.page_shift] * c.page_stride +
                                    kvh * c.head_stride + ((k + key) & page_mask) * c.slot_stride;
                const bool see = rg.sees(a, pos, k + key);
#pragma unroll
                for (int x = 0; x < DT32; ++x)
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const u32x2_t t = *reinterpret_cast<const u32x2_t *>(p + x * 32 + e * 2 + g * 4);
#pragma unroll
                        for (int z = 0; z < 4; ++z) {
                            const float o = odd_part<DT>(z & 1 ? t[z >> 1] >> 16 : t[z >> 1]);
                            acc[x][e + z] += see ? o : 0.f;
                        }
                    }
            }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int d = 0; d < DT32; ++d) {  // V^T operand: keys of step x, channels of tile d
                const int at = vbase + (((d * 4 + vch) ^ vx) << 4) + x * 16 * D * 2;
                const u32x2_t lo = tr_read(s_v[st], at), hi = tr_read(s_v[st], at + 8 * D * 2);
                acc[d] = mfma32<DT>((u32x4_t){lo.x, lo.y, hi.x, hi.y}, pf[x], acc[d]);
            }
        if (more) {
            ok = there(nxt);
            store(st ^ 1, i + 1, k2, ok);
        }
        k = k2;
        k2 = k3;
        nxt = nxt2;
        __syncthreads();
    }

    sum += __shfl_xor(sum, 32);
    if (!live) return;
    const int64_t row = static_cast<int64_t>(tok) * a.n_heads + head;
    if (a.pieces == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint16_t *o = a.out + row * D + g * 4;
#pragma unroll
        for (int x = 0; x < DT32; ++x)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                *reinterpret_cast<u32x2_t *>(o + x * 32 + e * 2) =
                    (u32x2_t){pack2<DT>(acc[x][e] * inv, acc[x][e + 1] * inv),
                              pack2<DT>(acc[x][e + 2] * inv, acc[x][e + 3] * inv)};
        if (a.lse && g == 0) a.lse[row] = sum == 0.f ? -INFINITY : m * kLn2 + logf(sum);
    } else {
        const int64_t at = row * a.pieces + part.first + piece;
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

// One workgroup per output row: O = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i over its
// pieces, in order; a piece that saw nothing has m_i = -inf and no O_i.
template <int DT, int D>
__global__ __launch_bounds__(D) void paged_attn_join_kernel(const Query a) {
    const int64_t row = blockIdx.x;
    const float2 *ml = a.part_ml + row * a.pieces;
    const float *o = a.part_o + row * a.pieces * D + threadIdx.x;
    float m = -INFINITY;
    for (int i = 0; i < a.pieces; ++i) m = fmaxf(m, ml[i].x);
    float l = 0.f, v = 0.f;
    for (int i = 0; i < a.pieces; ++i) {
        if (ml[i].x == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(ml[i].x - m);
        l += ml[i].y * f;
        v += o[static_cast<int64_t>(i) * D] * f;
    }
    a.out[row * D + threadIdx.x] = round16<DT>(l == 0.f ? 0.f : v / l);
    if (a.lse && threadIdx.x == 0) a.lse[row] = l == 0.f ? -INFINITY : m * kLn2 + logf(l);
}

// --------------------------------------------------------------------------------- host

int fill_cache(Cache &c, const nf4_paged_kv *kv, const int32_t *cu_q, int64_t tokens, int n_heads,
               int dtype) {
    if (!kv || (dtype != NF4_F16 && dtype != NF4_BF16)) return NF4_ERR_ARG;
    if (kv->pages < 0 || kv->page_size < 1 || kv->width < 0 || kv->batch < 0 || kv->n_kv < 1 ||
        tokens < 0 || n_heads < 1 || n_heads % kv->n_kv || kv->ld_table < kv->width)
        return NF4_ERR_ARG;
    // a position and a token times its heads stay 32-bit
    if (static_cast<int64_t>(kv->width) * kv->page_size > (1 << 30) || tokens > (1 << 26) ||
        n_heads > 1024 || kv->batch > (1 << 20))
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

// How a part runs: the kernel (rb row blocks of 16 in the few-rows kernel, 0 the tiled one), its
// items (sequences, or row blocks) and its pieces.
struct PartPlan {
    Part part;
    int rb, items;
};

struct Plan {
    PartPlan own, pre;
    int pieces;
    size_t bytes;
};

// `rows` rows at most of each of `items` sequences (prefix: items 1, the batch's rows) over
// `keys` keys at most.  Few rows go to the kernel without LDS staging; the tiles are cut until
// the launch has kFewGroups (kTileGroups) workgroups, or pieces of one slab a wave (4 tiles).
constexpr int kFewRows = 32, kFewGroups = 2048, kTileGroups = 512;

PartPlan plan_part(bool prefix, int64_t rows, int64_t blocks, int items, int n_kv, int64_t keys) {
    PartPlan p{};
    const bool few = rows <= kFewRows;
    p.rb = !few ? 0 : rows <= 16 ? 1 : 2;
    p.items = few ? (prefix ? 1 : items) : static_cast<int>(blocks);
    const int tiles = ceil_div(keys, few ? 32 : 64) + 1;
    const int64_t groups = static_cast<int64_t>(p.items) * n_kv;
    int64_t splits = (few ? kFewGroups : kTileGroups) / (groups ? groups : 1);
    splits = splits < 1 ? 1 : splits > ceil_div(tiles, 4) ? ceil_div(tiles, 4) : splits;
    const int per = ceil_div(ceil_div(tiles, splits), 4) * 4;
    p.part = Part{prefix ? 1 : 0, ceil_div(tiles, per), 0, per, static_cast<int>(blocks)};
    return p;
}

Plan make_plan(const Cache &c, int n_heads, int window, int sinks, int shared, int64_t max_q,
               int64_t max_len, int head_dim) {
    const int64_t group = n_heads / c.n_kv;
    int64_t longest = c.cu ? (max_q && max_q < c.tokens ? max_q : c.tokens) : c.uniform;
    const int64_t len = max_len && max_len < c.cap ? max_len : c.cap;
    int64_t span = len > shared ? len - shared : 0;
    if (window && span > static_cast<int64_t>(window) + longest + sinks) span = window + longest + sinks;
    const int seqs = c.batch + (c.cu ? 1 : 0);  // with offsets: and the tokens past the last
    const int64_t blocks = c.cu ? c.tokens * group / kRows + seqs
                                : static_cast<int64_t>(c.batch) * ceil_div(longest * group, kRows);
    Plan p{};
    p.own = plan_part(false, longest * group, blocks, seqs, c.n_kv, span);
    p.pieces = p.own.part.splits;
    if (shared) {
        const int64_t rows = c.tokens * group;
        p.pre = plan_part(true, rows, ceil_div(rows, kRows), 1, c.n_kv, len < shared ? len : shared);
        p.own.part.first = p.pre.part.splits;
        p.pieces += p.pre.part.splits;
    }
    if (p.pieces > 1)
        p.bytes = static_cast<size_t>(c.tokens) * n_heads * p.pieces * (4 * head_dim + 8);
    return p;
}

template <int DT, int D>
int launch_part(const Cache &c, const Query &a, const PartPlan &p, hipStream_t s) {
    const int64_t groups = static_cast<int64_t>(p.items) * p.part.splits * c.n_kv;
    if (groups == 0) return NF4_OK;
    if (groups > 0x7fffffff) return NF4_ERR_UNSUPPORTED;
    const dim3 grid(static_cast<unsigned>(groups));
    const bool small = c.page_shift < 4;
#define NF4_FEW(RB, SMALL)                                                                          \
    hipLaunchKernelGGL((paged_attn_few_kernel<DT, D, RB, SMALL>), grid, dim3(256), 0, s, c, a, p.part)
#define NF4_TILE(SMALL)                                                                             \
    hipLaunchKernelGGL((paged_attn_tile_kernel<DT, D, SMALL>), grid, dim3(256), 0, s, c, a, p.part)
    if (p.rb == 0) {
        if (small) NF4_TILE(true);
        else NF4_TILE(false);
    } else if (p.rb == 1) {
        if (small) NF4_FEW(1, true);
        else NF4_FEW(1, false);
    } else {
        if (small) NF4_FEW(2, true);
        else NF4_FEW(2, false);
    }
#undef NF4_FEW
#undef NF4_TILE
    return status_of(hipGetLastError());
}

template <int DT, int D>
int launch(const Cache &c, const Query &a, const Plan &p, hipStream_t s) {
    if (a.shared) {
        const int st = launch_part<DT, D>(c, a, p.pre, s);
        if (st != NF4_OK) return st;
    }
    const int st = launch_part<DT, D>(c, a, p.own, s);
    if (st != NF4_OK || p.pieces == 1) return st;
    hipLaunchKernelGGL((paged_attn_join_kernel<DT, D>), dim3(static_cast<unsigned>(c.tokens * a.n_heads)),
                       dim3(D), 0, s, a);
    return status_of(hipGetLastError());
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
    a.scale = fmaxf(fabsf(scale) * kLog2e, 1e-30f);  // not 0: a hidden score is -inf
    const Plan p = make_plan(c, n_heads, a.window, a.sinks, a.shared, max_q, max_len, kv->head_dim);
    a.pieces = p.pieces;
    if (p.bytes) {
        if (!workspace || workspace_bytes < p.bytes) return NF4_ERR_WORKSPACE;
        if (!aligned(workspace, 16)) return NF4_ERR_UNSUPPORTED;
        a.part_o = static_cast<float *>(workspace);
        a.part_ml = reinterpret_cast<float2 *>(a.part_o + tokens * n_heads * p.pieces * kv->head_dim);
    }
    auto s = static_cast<hipStream_t>(stream);
    const bool wide = kv->head_dim == 128;
    if (dtype == NF4_BF16)
        return wide ? launch<NF4_BF16, 128>(c, a, p, s) : launch<NF4_BF16, 64>(c, a, p, s);
    return wide ? launch<NF4_F16, 128>(c, a, p, s) : launch<NF4_F16, 64>(c, a, p, s);
}
