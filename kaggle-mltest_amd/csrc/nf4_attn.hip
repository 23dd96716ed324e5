// Attention of a packed training batch, forward and backward, for gfx950.
//
// Row i of sequence [s, e) sees keys j of [max(s, i - window + 1), i].  With t_ij = scale log2(e)
// q_i.k_j:   m_i = max_j t_ij,  l_i = sum_j 2^(t_ij - m_i),  P_ij = 2^(t_ij - m_i) / l_i,
//            o_i = sum_j P_ij v_j,
// and backward, from do and what the forward pass left (o, m, l), P formed again:
//            D_i = do_i.o_i,  dS_ij = P_ij (do_i.v_j - D_i),
//            dq_i = scale sum_j dS_ij k_j,  dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i P_ij do_i,
// the sums of dk and dv over the query heads that share the key too.  Offsets are device data, so
// every kernel bounds them itself.

#include "nf4_common.h"

#include <math.h>

#include <type_traits>

namespace {

struct Strided {  // [tokens, heads, D]: offsets in elements
    const uint16_t *p;
    int64_t tok, head;
    __device__ __forceinline__ const uint16_t *at(int t, int h) const { return p + t * tok + h * head; }
    __device__ __forceinline__ uint16_t *to(int t, int h) const { return const_cast<uint16_t *>(at(t, h)); }
};

struct Attn {
    Strided q, k, v, o, dout, dq, dk, dv;
    float2 *stats;  // [tokens][n_heads] (m, l)
    const int32_t *cu;
    int batch, tokens, window, n_heads, n_kv, group;
    float c;      // of the scores in units of log 2; not 0 (a hidden score is -inf)
    float scale;
};

// threadIdx.x, as the compiler does not know it: what is computed of it in a loop over tiles stays in there
// (ahead of the loop for two kinds of tiles at once, it took the registers that their own loops need).
__device__ __forceinline__ int thread_here() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// How many offsets are at or before t (the wave's), 64 at a time: a load's latency for every factor of
// 64 of the batch.
__device__ __forceinline__ int offsets_upto(const Attn &a, int t) {
    const int l = thread_here() & 63;
    int lo = 0, n = a.batch + 1;
    while (n > 64) {
        const int step = (n + 63) >> 6, i = l * step;
        const int c = __popcll(__ballot(i < n && a.cu[lo + i] <= t));
        if (c == 0) return lo;
        const int past = (c - 1) * step + 1;  // the offset c - 1 steps on is at or before t
        lo += past;
        n = n - past < step - 1 ? n - past : step - 1;
    }
    return lo + __popcll(__ballot(l < n && a.cu[lo + l] <= t));
}

// The rows [s, e) of the sequence of row t, or [t, t) of a row that belongs to none.  Every lane of the
// wave calls it, with rows of at most 32 from the first lane's on.
__device__ __forceinline__ int2 sequence_of(const Attn &a, int t) {
    if (!a.cu) return make_int2(0, a.tokens);
    // the next 64 offsets, a lane each, from the first row's sequence on
    const int i0 = offsets_upto(a, __builtin_amdgcn_readfirstlane(t)) - 1, l = thread_here() & 63;
    const int at = i0 + l < 0 ? 0 : i0 + l;
    const int next = at <= a.batch ? a.cu[at] : 0x7fffffff;
    int s = i0 < 0 ? 0x7fffffff : __builtin_amdgcn_readlane(next, 0), e = __builtin_amdgcn_readlane(next, 1);
    int k = 1;
    for (; k < 63 && __any(t >= e); ++k) {
        const int x = __builtin_amdgcn_readlane(next, k + 1);
        if (t >= e) {
            s = e;
            e = x;
        }
    }
    if (__any(t >= e)) {  // (more than 62 sequences in 32 rows: empty ones)
        int lo = 0, hi = a.batch + 1;  // the first offset past t
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.cu[mid] <= t) lo = mid + 1;
            else hi = mid;
        }
        s = lo == 0 ? 0x7fffffff : a.cu[lo - 1];
        e = lo > a.batch ? 0x7fffffff : a.cu[lo];
    }
    if (s > t || e <= t || e == 0x7fffffff) return make_int2(t, t);
    return make_int2(s < 0 ? 0 : s, e > a.tokens ? a.tokens : e);
}

// The keys [lo, hi) that row t sees, and the rows [t, hi) that see key t (t as above, or past the last
// row: none).
__device__ __forceinline__ int2 keys_of(const Attn &a, int t) {
    const int2 s = sequence_of(a, t < a.tokens ? t : a.tokens - 1);
    if (s.y <= t) return make_int2(t, t);
    return make_int2(a.window && t - a.window + 1 > s.x ? t - a.window + 1 : s.x, t + 1);
}
__device__ __forceinline__ int2 rows_of(const Attn &a, int t) {
    const int2 s = sequence_of(a, t < a.tokens ? t : a.tokens - 1);
    if (s.y <= t) return make_int2(t, t);
    return make_int2(t, a.window && t + a.window < s.y ? t + a.window : s.y);
}

// A score's exponent: fma(score, c, -m), exact but for its own rounding; where m is far from 0 the
// rounding of m itself would show in that (16 and more from 2^28 on), so there the product is rounded
// as m was.  It is above 0 by as much as m was rounded, which the row's sum has in it as well; a
// probability is at most 1 also where sums in another order would make more of it (`capped`).
constexpr float kFar = 1 << 20;
__device__ __forceinline__ float exponent(float s, float c, float m) {
    return fabsf(m) > kFar ? s * c - m : fmaf(s, c, -m);
}
__device__ __forceinline__ float capped(float x, float most) { return x > most ? most : x; }  // (a NaN stays)

// ------------------------------------------------------------------- one row, one key
//
// The definitions, a wave to a row or a key: fp32 throughout, nothing rounded on the way, and nothing
// read of what a row does not see.  Lanes take a key (or row) each for the dot products, then
// channels: lane l holds channels VE l .. VE l + VE - 1.

// x.y of two rows of D
template <int DT, int D>
__device__ __forceinline__ float dot_of(const uint16_t *x, const uint16_t *y) {
    float s = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; d += 8) {
        float a[8], b[8];
        unpack8<DT>(*reinterpret_cast<const u32x4_t *>(x + d), a);
        unpack8<DT>(*reinterpret_cast<const u32x4_t *>(y + d), b);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(a[i], b[i], s);
    }
    return s;
}

__device__ __forceinline__ float lane_value(float v, int l) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}

// this lane's channels of a row (one in the low half, where it holds one)
template <int D>
__device__ __forceinline__ uint32_t channels_of(const uint16_t *row) {
    const int l = thread_here() & 63;
    if constexpr (D == 128) return *reinterpret_cast<const uint32_t *>(row + 2 * l);
    else return row[l];
}
// acc += f * them
template <int DT, int D>
__device__ __forceinline__ void add_channels(float (&acc)[D / 64], float f, uint32_t w) {
    acc[0] = fmaf(f, f32_of<DT>(w & 0xffffu), acc[0]);
    if constexpr (D == 128) acc[1] = fmaf(f, f32_of<DT>(w >> 16), acc[1]);
}
template <int DT, int D>
__device__ __forceinline__ void add_row(float (&acc)[D / 64], float f, const uint16_t *row) {
    add_channels<DT, D>(acc, f, channels_of<D>(row));
}

template <int DT, int D>
__device__ __forceinline__ void store_row(uint16_t *row, const float (&v)[D / 64]) {
    const int l = thread_here() & 63;
    if constexpr (D == 128)
        *reinterpret_cast<uint32_t *>(row + 2 * l) = round16<DT>(v[0]) | static_cast<uint32_t>(round16<DT>(v[1])) << 16;
    else row[l] = round16<DT>(v[0]);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// acc = sum over keys [k0, k1) of 2^(t - m) v, of row r whose largest t is m; rows of v are asked for some
// at a time
constexpr int kAtOnce = 16;
template <int DT, int D>
__device__ __forceinline__ void row_forward(const Attn &a, int head, int r, int k0, int k1, float m,
                                            float (&acc)[D / 64]) {
    const int lane = thread_here() & 63, kvh = head / a.group;
    const uint16_t *q = a.q.at(r, head);
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] = 0.f;
    for (int k = k0; k < k1; k += 64) {
        float p = 0.f;
        if (k + lane < k1)
            p = __builtin_amdgcn_exp2f(exponent(dot_of<DT, D>(q, a.k.at(k + lane, kvh)), a.c, m));
        const int n = k1 - k < 64 ? k1 - k : 64;
        for (int i = 0; i < n; i += kAtOnce) {
            uint32_t w[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) w[u] = channels_of<D>(a.v.at(k + (i + u < n ? i + u : n - 1), kvh));
#pragma unroll
            for (int u = 0; u < kAtOnce && i + u < n; ++u) add_channels<DT, D>(acc, lane_value(p, i + u), w[u]);
        }
    }
}

// acc = sum over keys [k0, k1) of dS k
template <int DT, int D>
__device__ __forceinline__ void row_backward(const Attn &a, int head, int r, int k0, int k1,
                                             float (&acc)[D / 64]) {
    const int lane = thread_here() & 63, kvh = head / a.group;
    const uint16_t *q = a.q.at(r, head), *go = a.dout.at(r, head);
    const float2 ml = a.stats[static_cast<int64_t>(r) * a.n_heads + head];
    const float delta = dot_of<DT, D>(go, a.o.at(r, head)), inv = 1.f / ml.y;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] = 0.f;
    for (int k = k0; k < k1; k += 64) {
        float ds = 0.f;
        if (k + lane < k1) {
            const float p = capped(__builtin_amdgcn_exp2f(exponent(dot_of<DT, D>(q, a.k.at(k + lane, kvh)), a.c, ml.x)) * inv, 1.f);
            ds = p * (dot_of<DT, D>(go, a.v.at(k + lane, kvh)) - delta);
        }
        const int n = k1 - k < 64 ? k1 - k : 64;
        for (int i = 0; i < n; ++i) add_row<DT, D>(acc, lane_value(ds, i), a.k.at(k + i, kvh));
    }
}

// dk += sum over rows [r0, r1) of dS q, dv += sum P do, of key j and query head `head`
template <int DT, int D>
__device__ __forceinline__ void key_backward(const Attn &a, int head, int j, int r0, int r1,
                                             float (&dk)[D / 64], float (&dv)[D / 64]) {
    const int lane = thread_here() & 63, kvh = head / a.group;
    const uint16_t *kj = a.k.at(j, kvh), *vj = a.v.at(j, kvh);
    for (int r = r0; r < r1; r += 64) {
        float p = 0.f, ds = 0.f;
        if (r + lane < r1) {
            const float2 ml = a.stats[static_cast<int64_t>(r + lane) * a.n_heads + head];
            const uint16_t *go = a.dout.at(r + lane, head);
            p = capped(__builtin_amdgcn_exp2f(exponent(dot_of<DT, D>(kj, a.q.at(r + lane, head)), a.c, ml.x)) / ml.y, 1.f);
            ds = p * (dot_of<DT, D>(vj, go) - dot_of<DT, D>(go, a.o.at(r + lane, head)));
        }
        const int n = r1 - r < 64 ? r1 - r : 64;
        for (int i = 0; i < n; ++i) {
            add_row<DT, D>(dv, lane_value(p, i), a.dout.at(r + i, head));
            add_row<DT, D>(dk, lane_value(ds, i), a.q.at(r + i, head));
        }
    }
}

// --------------------------------------------------------------------------- tiles
//
// A workgroup of four waves owns 128 rows (or keys), 32 a wave, in registers, and goes over the keys (or
// rows) that they see in tiles of 64, which come to LDS by DMA while the tile before is used (two
// stages, one barrier a tile).  The first products are formed so that a lane holds one of its own
// rows (a column of the MFMA result): what belongs to a row stays in the lane, and the probabilities
// leave the first product in the register layout that the second takes as its operand.
//
// 16-byte chunk ch of a tile's row r lies at chunk ch ^ swizzle(r): the 16 lanes that LDS serves at a
// time read one chunk of 16 rows from 16 bank groups, and 64 bytes of each of 4 consecutive rows
// (transposed reads) from all banks.

constexpr int kOwn = 128, kTile = 64, kRows = 32;  // (kRows: a tile of rows in the backward pass)

template <int D>
__device__ __forceinline__ constexpr int swizzle(int r) {
    return D == 128 ? (r & 3) << 2 | (r >> 2 & 3) : (r & 2) << 1 | (r >> 2 & 3);
}

template <int D>
constexpr int kTileBytes = kTile * D * 2;

// A tensor's tiles of ROWS rows of a head, one after the other: where the next begins, and what a thread
// knows of them: the byte of its 16 in the first pass, and the passes' distance.
template <int D, int ROWS>
struct Stager {
    static constexpr int CH = D / 8, RPP = 256 / CH;
    const uint16_t *next;
    int pitch, off;  // bytes

    __device__ __forceinline__ void begin(const Strided &x, int head, int t) {
        next = reinterpret_cast<const uint16_t *>(uniform64(reinterpret_cast<int64_t>(x.p + head * x.head + t * x.tok)));
    }
    __device__ __forceinline__ void set(const Strided &x, int head, int t, int tid) {
        const int row = tid / CH, ch = tid % CH;
        begin(x, head, t);
        pitch = static_cast<int>(x.tok) * 2;
        off = row * pitch + ((ch ^ swizzle<D>(row)) << 4);
    }
    // the next tile to LDS address `at` (the wave's); rows from `rows` on, and the first `skip`, are zeros, and not
    // read (the buffer begins at row `skip`: offsets before it are negative, which is past its end)
    __device__ __forceinline__ void send(uint32_t at, int rows, int skip = 0) {
        const int n = (rows < ROWS ? rows : ROWS) - skip, before = skip * pitch;
        const auto *first = reinterpret_cast<const char *>(next) + before;
        const rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(first), static_cast<short>(0),
                                                           n > 0 ? (n - 1) * pitch + D * 2 : 0, 0x00020000);
#pragma unroll
        for (int x = 0; x < ROWS / RPP; ++x) lds_dma16(at + x * 4096, off + x * RPP * pitch - before, r, 0);
        next = reinterpret_cast<const uint16_t *>(reinterpret_cast<const char *>(next) + static_cast<int64_t>(ROWS) * pitch);
    }
};

// Operand addresses of a lane in a tile at LDS address 0: rows as they lie (a row a lane, 16 channels
// a step), and transposed (a channel a lane, 16 rows a step).
template <int D>
__device__ __forceinline__ uint32_t row_address(int l) {
    const int n = l & 31, g = l >> 5;
    return n * D * 2 + ((g ^ swizzle<D>(n)) << 4);
}
template <int D>
__device__ __forceinline__ uint32_t channel_address(int l) {
    const int row = (l >> 5) * 4 + ((l & 15) >> 2);
    const int ch = ((l >> 4) & 1) * 2 + ((l & 3) >> 1);
    return row * D * 2 + (l & 1) * 8 + ((ch ^ swizzle<D>(row)) << 4);
}
// channels 16 x .. of rows 32 h .. of the tile at `at`
template <int D>
__device__ __forceinline__ u32x4_t rows_operand(uint32_t at, int h, int x) {
    return lds16((at ^ (x << 5)) + h * 64 * D);
}
// rows 16 x .. (in the order of a result's registers) of channels 32 d ..
template <int D>
__device__ __forceinline__ u32x4_t channels_operand(uint32_t at, int x, int d) {
    const uint32_t p = at ^ (d << 6);
    const u32x2_t lo = tr_read(p + x * 32 * D), hi = tr_read((p ^ 32) + x * 32 * D + 16 * D);
    return (u32x4_t){lo.x, lo.y, hi.x, hi.y};
}

// A lane's own row as operands: channels 16 x + 8 (l / 32) ..
template <int D>
__device__ __forceinline__ void own_operand(u32x4_t (&f)[D / 16], const uint16_t *row, bool live, int l,
                                            uint32_t flip = 0) {
    const int g = l >> 5;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
        f[x] = (u32x4_t){0, 0, 0, 0};
        if (live) f[x] = *reinterpret_cast<const u32x4_t *>(row + x * 16 + g * 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[x][i] ^= flip;
    }
}

// The registers of a result, as 16-bit operands of the next product (x: 16 of its 32 rows).
template <int DT>
__device__ __forceinline__ u32x4_t operand_of(const float16_t &v, int x) {
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = pack2<DT>(v[x * 8 + 2 * i], v[x * 8 + 2 * i + 1]);
    return r;
}

// What the rows (or keys) of a wave and of a workgroup see: [lo, hi) any of them, [full_lo, full_hi)
// all of them (empty ones apart).  Both ends grow with the row, so the first and the last that see
// anything tell; with offsets that decrease some see less than they would, and nothing out of range.
struct Span {
    int lo, hi, full_lo, full_hi;
    __device__ __forceinline__ void set(int2 s) {
        const uint64_t some = __ballot(s.x < s.y);
        const int first = some ? __builtin_ctzll(some) : 0;
        const int last = (some & 0xffffffffull) ? 31 - __builtin_clz(static_cast<uint32_t>(some)) : 0;
        lo = some ? __builtin_amdgcn_readlane(s.x, first) : 0x7fffffff;
        hi = some ? __builtin_amdgcn_readlane(s.y, last) : 0;
        full_lo = __builtin_amdgcn_readlane(s.x, last);
        full_hi = __builtin_amdgcn_readlane(s.y, first);
    }
    // over the four waves; `mem`: 8 words of LDS
    __device__ __forceinline__ int2 all(int *mem) const {
        const int w = threadIdx.x >> 6;
        if ((thread_here() & 63) == 0) {
            mem[w] = lo;
            mem[4 + w] = hi;
        }
        __syncthreads();
        int a = mem[0], b = mem[4];
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            a = mem[i] < a ? mem[i] : a;
            b = mem[4 + i] > b ? mem[4 + i] : b;
        }
        return make_int2(__builtin_amdgcn_readfirstlane(a), __builtin_amdgcn_readfirstlane(b));
    }
    __device__ __forceinline__ bool full(int t, int n) const { return t >= full_lo && t + n <= full_hi; }
    __device__ __forceinline__ bool none(int t, int n) const { return t >= hi || t + n <= lo; }
};

// The bits of a 64-wide tile at t that are in [s.x, s.y), for this lane's registers: register e of
// half h is bit 32 h + 8 (e / 4) + e % 4.
__device__ __forceinline__ uint64_t seen_bits(int2 s, int t) {
    return (below(s.y - t) & ~below(s.x - t)) >> (((thread_here() >> 5) & 1) * 4);
}
__device__ __forceinline__ bool bit_of(uint64_t m, int h, int e) {
    return static_cast<uint32_t>(m >> (32 * h)) >> (8 * (e >> 2) + (e & 3)) & 1;
}

// Probabilities, and dS in the backward pass, are rounded to the inputs' 16 bits for the second product, half a
// step each: they are operands of matrix instructions, which take fp32 at a sixteenth of the rate.  Against 64
// bits, results are off by 1.1 (forward) to 1.4 times (backward) as much as with fp32 in their place, rounded once
// at the end.  fp16's probabilities are 2^15 times as large, so that those down to 2^-29 keep their bits (its
// least normal number is 2^-14).
template <int DT>
constexpr float kTop = DT == NF4_BF16 ? 0.f : 15.f;

// Infinities and NaN.  A probability of 0 that stands for a key that is not seen makes NaN of an infinity
// or NaN beside it in the tile.  So a row (or key) whose sums hold a NaN is formed again from what it
// sees alone, by the functions above, unless what it sees says that it is NaN.  That takes 50 us for a row of 2000
// keys, one behind the other: it is for the rows (or keys) that share a workgroup's 128 with some that see the
// value, and what no row of a workgroup sees comes to LDS as zeros.
template <int N>
__device__ __forceinline__ bool any_nan(const float16_t (&v)[N]) {
    float odd = 0.f;
#pragma unroll
    for (int x = 0; x < N; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) odd = fmaf(v[x][e], 0.f, odd);
    bool z = false;
    if (__any(odd != 0.f)) {  // (one instruction a register, where all are finite)
#pragma unroll
        for (int x = 0; x < N; ++x)
#pragma unroll
            for (int e = 0; e < 16; ++e) z |= v[x][e] != v[x][e];
    }
    return z;
}
// the rows of a wave (bit n: lanes n and n + 32) for which `which` is true of a lane
__device__ __forceinline__ uint32_t rows_where(bool which) {
    const uint64_t m = __ballot(which);
    return static_cast<uint32_t>(m) | static_cast<uint32_t>(m >> 32);
}
template <int N>
__device__ __forceinline__ void fill_of(float16_t (&v)[N], float f) {
#pragma unroll
    for (int x = 0; x < N; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) v[x][e] = f;
}

// Which of a wave's rows (bits) see a value x [keys, D] that makes its sum NaN, for each of a lane's channels
// D / 64 l ..: a NaN of v in the forward pass, with INFS also an infinity, of k in the backward pass (a row that is
// not NaN itself has a score of -inf with such a key, and 0 times an infinity in that channel).  `seen`: the
// keys of this lane's row; all rows' lie in [lo, hi).  One pass over x for the 32 rows; formed again one by one, all
// rows behind an early NaN of v made the forward pass 110 times as long at 2048 tokens, 280 times at 4096, and those
// behind an infinite k the backward pass 40 and 60 times.
template <int DT, int D, bool INFS>
__device__ __forceinline__ void nan_by(const Strided &v, int head, int lo, int hi, int2 seen, uint32_t (&by)[D / 64]) {
    constexpr uint32_t MOST = (DT == NF4_BF16 ? 0x7f80u : 0x7c00u) - INFS;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) by[i] = 0;
    for (int k = lo; k < hi; k += kAtOnce) {
        uint32_t w[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) w[u] = channels_of<D>(v.at(k + u < hi ? k + u : hi - 1, head));
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const bool x = (w[u] & 0x7fffu) > MOST, y = D == 128 && (w[u] >> 16 & 0x7fffu) > MOST;
            if (!__any(x || y)) continue;
            const uint32_t rows = rows_where(seen.x <= k + u && k + u < seen.y);
            if (x) by[0] |= rows;
            if (y) by[D / 64 - 1] |= rows;
        }
    }
}
// A NaN of this lane's row in a channel for which `by` does not name the row.
template <int D>
__device__ __forceinline__ bool unexplained(const float16_t (&v)[D / 32], const uint32_t (&by)[D / 64]) {
    const int l = thread_here() & 63;
    bool z = false;
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int c = x * 32 + 8 * (e >> 2) + 4 * (l >> 5) + (e & 3);  // (c and e are odd together)
            const uint32_t rows = __shfl(by[e % (D / 64)], c / (D / 64));
            z |= v[x][e] != v[x][e] && !(rows >> (l & 31) & 1);
        }
    return z;
}

// This lane's channels of its row, from a transposed result.
template <int DT, int D>
__device__ __forceinline__ void store_own(uint16_t *row, const float16_t (&v)[D / 32], float f) {
    row += ((thread_here() & 63) >> 5) * 4;
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<u32x2_t *>(row + x * 32 + e * 2) =
                (u32x2_t){pack2<DT>(v[x][e] * f, v[x][e + 1] * f), pack2<DT>(v[x][e + 2] * f, v[x][e + 3] * f)};
}

// An output is a mean of values: one past fp16's last number is there by the roundings of its
// probabilities (a step at most), and is that number.
template <int DT, int N>
__device__ __forceinline__ void keep_finite(float16_t (&v)[N], float f) {
    if constexpr (DT == NF4_F16) {
#pragma unroll
        for (int x = 0; x < N; ++x)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                v[x][e] *= f;
                v[x][e] = fabsf(v[x][e]) < INFINITY ? __builtin_amdgcn_fmed3f(v[x][e], -65504.f, 65504.f) : v[x][e];
            }
    }
}

// Pieces.  Where a launch has too few tiles to fill the card, or they are too uneven, what a tile of
// rows (or keys) goes over is cut into pieces of `per` steps, a workgroup each; what a piece leaves is
// fp32 in `part`, and the join launch sums a tile's pieces in their order.  A tile in one piece writes
// its result itself.
struct Pieces {
    int per, most;  // steps of a piece, at least; pieces of a tile, at most
    float *part;    // [tiles * heads][most][arrays][4 waves][32 D]
    float2 *ml;     // forward: [tiles * heads][most][128]
    __device__ __forceinline__ int of(int n) const {
        const int p = (n + per - 1) / per;
        return p < 1 ? 1 : p < most ? p : most;
    }
};

// Steps of UNIT that a tile's rows (or keys) go over, found by four waves of 32 of its rows.
template <int UNIT>
__device__ __forceinline__ int steps_of_tile(const Attn &a, int tile, bool of_rows, int *mem) {
    const int t = tile * kOwn + (threadIdx.x >> 6) * 32 + (threadIdx.x & 31);
    Span sp;
    sp.set(of_rows ? keys_of(a, t) : rows_of(a, t));
    const int2 all = sp.all(mem);
    return all.x < all.y ? (all.y - 1) / UNIT - all.x / UNIT + 1 : 0;
}

// Steps [x, y) of piece i of p.
__device__ __forceinline__ int2 steps_of(int n, int p, int i) {
    const int per = (n + p - 1) / p, x = i * per;
    return make_int2(x < n ? x : n, x + per < n ? x + per : n);
}

// The 32 rows of a wave in `part`: its registers as they are, 16 bytes a lane one behind the other
// (as rows of D, 64 lanes write 64 lines at a time: a join of 280 pieces 23 us instead of 16).
template <int D>
__device__ __forceinline__ void store_part(float *part, const float16_t (&v)[D / 32]) {
    part += (thread_here() & 63) * 4;
#pragma unroll
    for (int x = 0; x < D / 32; ++x)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
            *reinterpret_cast<float4_t *>(part + (x * 4 + e / 4) * 256) = (float4_t){v[x][e], v[x][e + 1], v[x][e + 2], v[x][e + 3]};
}
// row i of them, VE channels a lane
template <int D>
__device__ __forceinline__ void store_part_row(float *part, int i, const float (&v)[D / 64]) {
#pragma unroll
    for (int x = 0; x < D / 64; ++x) {
        const int c = (thread_here() & 63) * (D / 64) + x;
        part[(c >> 3) * 256 + ((c >> 2 & 1) * 32 + i) * 4 + (c & 3)] = v[x];
    }
}
// The sums of the pieces' rows go to memory through LDS ([32][D + 8]), a row's 16 bytes a thread.
template <int DT, int D>
__device__ __forceinline__ void join_put(uint16_t *lds, int i, const float4_t &v) {  // float4 i of a wave's
    const int lane = i & 63;
    *reinterpret_cast<u32x2_t *>(lds + (lane & 31) * (D + 8) + (i >> 6) * 8 + (lane >> 5) * 4) =
        (u32x2_t){pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
}
template <int D>
__device__ __forceinline__ void join_write(const Strided &out, int head, int r0, int tokens, const uint16_t *lds) {
    __syncthreads();
#pragma unroll
    for (int x = threadIdx.x; x < 4 * D; x += 256) {
        const int i = x / (D / 8), ch = x % (D / 8) * 8;
        if (r0 + i < tokens)
            *reinterpret_cast<u32x4_t *>(out.to(r0 + i, head) + ch) = *reinterpret_cast<const u32x4_t *>(lds + i * (D + 8) + ch);
    }
}

// ------------------------------------------------------------------------------ forward
//
// The running maximum and sum of a row stay in its lane; a wave whose rows' maxima all hold does not rescale.  8192
// tokens of 28 heads of 128 over 4, bf16: 490-512 us from card to card, 940-980 TFLOP/s.  A step of 64 keys for 128
// rows takes two workgroups on a CU 2.2 us.  In a loop of its own it takes 1.98: its matrix instructions alone, on
// values as these are, 1.27 at the clock that the power cap leaves (0.93 on zeros), the exponentials, maxima and
// sums 0.24 more, reading k and v out of LDS 0.27, barrier and DMA 0.2; where the other 0.2 go was not found.  8192
// tokens of 14 heads of 64 over 2, bf16: 181 us; a lane has as many exponentials for half the products, and its
// vector instructions take about three quarters of the cycles.  (The next step's scores formed between this one's
// exponentials, in the same wave: 20 % slower, and not faster without its spills, in steps of 32 keys.)
template <int DT, int D>
__global__ __launch_bounds__(256, 2) void attn_fwd_kernel(const Attn a, const Pieces pc, int tiles) {
    constexpr int KS = D / 16, DN = D / 32, TB = kTileBytes<D>;
    __shared__ __attribute__((aligned(16))) uint8_t lds[4 * TB + 64];
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & 63;
    const int g = l >> 5, n = l & 31;
    const int piece = blockIdx.x / (tiles * a.n_heads), block = blockIdx.x % (tiles * a.n_heads);
    const int kvh = block % a.n_kv, y = block / a.n_kv;
    const int head = kvh * a.group + y % a.group;
    const int tile = tiles - 1 - y / a.group;  // (the last rows see most: first)
    const int r = tile * kOwn + w * 32 + n;
    const int2 seen = keys_of(a, r);
    Span sp;
    sp.set(seen);
    int2 all = sp.all(reinterpret_cast<int *>(lds + 4 * TB));
    const int k0 = all.x & ~(kTile - 1), steps = all.x < all.y ? (all.y - k0 + kTile - 1) / kTile : 0;
    const int pieces = pc.of(steps);
    if (piece >= pieces) return;
    const int2 mine_of = steps_of(steps, pieces, piece);
    const int k1 = k0 + mine_of.y * kTile;  // (past the last key in the last piece)
    all.y = k1 < all.y ? k1 : all.y;

    u32x4_t q[KS];
    const float c = fabsf(a.c);
    own_operand<D>(q, a.q.at(r, head), r < a.tokens, l, a.c < 0.f ? 0x80008000u : 0u);
    Stager<D, kTile> sk, sv;
    const int first = k0 + mine_of.x * kTile;
    sk.set(a.k, kvh, first, threadIdx.x);
    sv.set(a.v, kvh, first, threadIdx.x);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) uint8_t *)lds));
    const uint32_t mine = __builtin_amdgcn_readfirstlane(lds0 + w * 1024);
    const uint32_t ka = lds0 + row_address<D>(l), va = lds0 + 2 * TB + channel_address<D>(l);

    float m = -INFINITY, sum = 0.f;
    bool far = false;  // a row's m is (of the wave's; each row by its own, as in the backward pass)
    float16_t acc[DN];
#pragma unroll
    for (int x = 0; x < DN; ++x) acc[x] = (float16_t){};
    int k = steps ? first : all.y, st = 0;
    if (k < all.y) {
        // (what lies before the rows' first key is not theirs: with a NaN in it every one of their sequence's
        // rows was formed again)
        const int skip = all.x > k ? all.x - k : 0;
        sk.send(mine, all.y - k, skip);
        sv.send(mine + 2 * TB, all.y - k, skip);
    }
    for (; k < all.y; k += kTile, st ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();  // every wave's part of this tile is there, and the one before is read
        if (k + kTile < all.y) {
            sk.send(mine + (st ^ 1) * TB, all.y - k - kTile);
            sv.send(mine + (2 + (st ^ 1)) * TB, all.y - k - kTile);
        }
        if (sp.none(k, kTile)) continue;
        u32x4_t kf[2][KS];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int x = 0; x < KS; ++x) kf[h][x] = rows_operand<D>(ka + st * TB, h, x);
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
        float16_t sc[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sc[h] = (float16_t){};
#pragma unroll
            for (int x = 0; x < KS; ++x) sc[h] = mfma32<DT>(kf[h][x], q[x], sc[h]);
        }
        __builtin_amdgcn_s_setprio(0);
        u32x4_t vf[2][DN];
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int d = 0; d < DN; ++d) vf[x][d] = channels_operand<D>(va + st * TB, x, d);
        __builtin_amdgcn_sched_barrier(0);
        if (!sp.full(k, kTile)) {
            const uint64_t see = seen_bits(seen, k);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!bit_of(see, h, e)) sc[h][e] = -INFINITY;
        }
        float top = sc[0][0];
#pragma unroll
        for (int e = 1; e < 32; ++e) top = fmaxf(top, sc[e >> 4][e & 15]);
        const float t = fmaxf(top, other_half(top)) * c;
        const float mn = fmaxf(m, fabsf(t) > kFar ? t : t - kTop<DT>);
        if (__any(mn > m)) {
            const float alpha = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
            sum *= alpha;
#pragma unroll
            for (int x = 0; x < DN; ++x) acc[x] *= alpha;
            m = mn;
            far = __any(fabsf(m) > kFar && m != -INFINITY);
        }
        const float base = m == -INFINITY ? 0.f : m;
        if (__builtin_expect(far, 0)) {
#pragma unroll
            for (int e = 0; e < 32; ++e) sc[e >> 4][e & 15] = exponent(sc[e >> 4][e & 15], c, base);
        }
        const float mul = far ? 1.f : c, sub = far ? 0.f : base;
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[e >> 4][e & 15], mul, -sub));
            sum += p;
            sc[e >> 4][e & 15] = p;
        }
        u32x4_t pf[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) pf[x] = operand_of<DT>(sc[x >> 1], x & 1);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
#pragma unroll
            for (int d = 0; d < DN; ++d) acc[d] = mfma32<DT>(vf[x & 1][d], pf[x], acc[d]);
            if (x < 2)
#pragma unroll
                for (int d = 0; d < DN; ++d) vf[x][d] = channels_operand<D>(va + st * TB, x + 2, d);
        }
        __builtin_amdgcn_s_setprio(0);
    }

    sum += other_half(sum);
    const int2 part = make_int2(seen.x > first ? seen.x : first, seen.y < all.y ? seen.y : all.y);  // of this piece
    const bool some = part.x < part.y;
    const int64_t slot = ((static_cast<int64_t>(tile) * a.n_heads + head) * pc.most + piece) * kOwn + w * 32;
    const bool nan = some && !(sum > 0.f && fabsf(m) < INFINITY);  // a score is NaN or +inf, or all are -inf
    const bool none = nan && pieces > 1 && m == -INFINITY && sum == 0.f;  // (here: other pieces may have more)
    uint32_t again = rows_where(some && !nan && any_nan(acc));
    if (again) {  // but for what a NaN of v explains
        uint32_t by[D / 64];
        nan_by<DT, D, false>(a.v, kvh, sp.lo > first ? sp.lo : first, sp.hi < all.y ? sp.hi : all.y, part, by);
        again &= rows_where(unexplained<D>(acc, by));
    }
    // a row that sees nothing has zeros (its registers hold anything: no mask kept tiles from it that every
    // other row of its wave sees whole)
    if (!some || none) fill_of(acc, 0.f);
    else if (nan) fill_of(acc, NAN);
    const bool f = fabsf(m) > kFar;
    float2 ml = make_float2(f ? m : m + kTop<DT>, f ? sum : __builtin_amdgcn_ldexpf(sum, -static_cast<int>(kTop<DT>)));
    if (nan) ml = none ? make_float2(m, 0.f) : make_float2(NAN, NAN);
    if (!some) ml = make_float2(0.f, 0.f);
    const bool mine_now = r < a.tokens && !(again >> n & 1);
    if (pieces == 1 && r < a.tokens && g == 0) a.stats[static_cast<int64_t>(r) * a.n_heads + head] = ml;
    if (pieces > 1) {
        if (!f && some)
#pragma unroll
            for (int x = 0; x < DN; ++x) acc[x] *= __builtin_amdgcn_ldexpf(1.f, -static_cast<int>(kTop<DT>));
        store_part<D>(pc.part + slot * D, acc);  // (rows that follow below or are not there, too)
        if (g == 0) pc.ml[slot + n] = ml;
    } else if (mine_now) {
        const float inv = some ? 1.f / sum : 0.f;
        keep_finite<DT>(acc, inv);
        store_own<DT, D>(a.o.to(r, head), acc, DT == NF4_F16 ? 1.f : inv);
    }
    if (!again) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (parts are there before their rows are written again)
#pragma unroll 1
    for (uint32_t left = again; left; left &= left - 1) {
        const int i = __builtin_ctz(left), row = tile * kOwn + w * 32 + i;
        float o[D / 64];
        row_forward<DT, D>(a, head, row, __builtin_amdgcn_readlane(part.x, i), __builtin_amdgcn_readlane(part.y, i),
                           lane_value(ml.x, i), o);
        if (pieces > 1) {
            store_part_row<D>(pc.part + slot * D, i, o);
            continue;
        }
        const float rl = lane_value(ml.y, i);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) o[x] /= rl;
        store_row<DT, D>(a.o.to(row, head), o);
    }
}

// A workgroup joins 32 rows of a tile that is in pieces: each a (m, l, o) of its keys.
template <int DT, int D>
__global__ __launch_bounds__(256) void attn_fwd_join_kernel(const Attn a, const Pieces pc) {
    __shared__ __attribute__((aligned(16))) uint16_t lds[32 * (D + 8)];
    __shared__ int mem[8];
    const int tile = blockIdx.x >> 2, w = blockIdx.x & 3, head = blockIdx.y;
    const int pieces = pc.of(steps_of_tile<kTile>(a, tile, true, mem));
    if (pieces < 2) return;
    const int64_t slot = (static_cast<int64_t>(tile) * a.n_heads + head) * pc.most * kOwn + w * 32;
    const int n = threadIdx.x & 31, r = tile * kOwn + w * 32 + n;
    float m = -INFINITY, l = 0.f;
    if (r < a.tokens) {
        bool all_low = false;  // a piece saw scores of -inf only
        for (int p = 0; p < pieces; ++p) {
            const float2 x = pc.ml[slot + p * kOwn + n];
            if (x.y != 0.f) m = fmaxf(m, x.x);  // (0: it saw nothing)
            else all_low |= x.x == -INFINITY;
        }
        for (int p = 0; p < pieces; ++p) {
            const float2 x = pc.ml[slot + p * kOwn + n];
            if (x.y != 0.f) l += x.y * (x.x == m ? 1.f : __builtin_amdgcn_exp2f(x.x - m));
        }
        if (l == 0.f && all_low) l = NAN;
        if (threadIdx.x < 32)
            a.stats[static_cast<int64_t>(r) * a.n_heads + head] = l == 0.f ? make_float2(0.f, 0.f) : make_float2(l == l ? m : NAN, l);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    float4_t o[D / 32];
#pragma unroll
    for (int x = 0; x < D / 32; ++x) o[x] = (float4_t){0.f, 0.f, 0.f, 0.f};
    if (r < a.tokens)
        for (int p = 0; p < pieces; ++p) {
            const float2 x = pc.ml[slot + p * kOwn + n];
            if (x.y == 0.f) continue;
            const float f = (x.x == m ? 1.f : __builtin_amdgcn_exp2f(x.x - m)) * inv;
            const float *part = pc.part + (slot + p * kOwn) * D + threadIdx.x * 4;
#pragma unroll
            for (int y = 0; y < D / 32; ++y) o[y] += *reinterpret_cast<const float4_t *>(part + y * 1024) * f;
        }
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
        if constexpr (DT == NF4_F16)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[x][e] = fabsf(o[x][e]) < INFINITY ? __builtin_amdgcn_fmed3f(o[x][e], -65504.f, 65504.f) : o[x][e];
        if (l != l) o[x] = (float4_t){NAN, NAN, NAN, NAN};
        join_put<DT, D>(lds, x * 256 + threadIdx.x, o[x]);
    }
    join_write<D>(a.o, head, tile * kOwn + w * 32, a.tokens, lds);
}

// ----------------------------------------------------------------------------- backward
//
// What the backward pass reads of a row for every key, in blocks of 32 rows, four numbers each: m,
// log2 l and m + log2 l (in fp16 less kTop), and -D; zeros of a row of no sequence, and NaN of a row whose
// do, statistics or D hold an infinity or NaN: its dq is NaN then, and the dk and dv of every key that it
// sees (elementwise some would be infinite or finite; that costs what forming them one by one does, and a
// loss whose scale was too high has such rows everywhere).  Where |m| is below kNear a probability's exponent
// is taken with the sum of the first two, whose rounding (2^-16) is below those that follow.
constexpr float kNear = 256.f;

// Tiles or shares.  Where all tiles are short, each has a workgroup.  Else that is uneven, and a
// key/value head's work is a line: its tiles of keys one behind the other, then the tiles of rows of its
// query heads, each as long as its steps cost and its beginning.  `groups` workgroups take an equal share
// of the line each, which may begin and end inside a tile: all are on the card at once and end together,
// whatever the lengths of the sequences are (device data).  A step belongs to the share in which it
// begins; a tile whose steps are in several leaves a part for each, and the join launch sums a tile's
// parts in their order.  (Heads of 128, bf16, the whole pass: one sequence of 2048, 12 heads over 2: 81 us,
// a fifth more with pieces of equal length; of 4096: 210, 28 % more; of 8192, 28 over 4: 1640, the same; 30
// sequences of 200, 16 heads of 64: 50 with a workgroup a tile, 40 % more with shares.  Half as many shares,
// one a CU: 2048 100 us, 8192 2270.)
//
// What bounds it, bf16, 8192 tokens of 28 heads of 128 over 4: the rows' launch 22 us, this one about 1600, the
// join 22; 1590-1730 together, from card to card.  It does 7 products where a formula's 5 would do (the scores and
// do.v are formed for the keys and for the rows again, since a sum of dq over the keys' workgroups would need
// atomics, whose order changes results): 1.04 PFLOP/s of them, where a large matrix product by the library reaches
// 1.35.  The matrix pipe is busy 51 % of the cycles, at 1.64 GHz: the power cap.  At 2048 tokens of 12 heads (65
// us, the join 15) a workgroup has about 17 steps, and 55 MB of parts are written and read again.  Both bodies, the
// rows and keys formed one by one and the shares' bookkeeping are one kernel: with heads of 128 it has all 256
// vector registers (bf16 two more, in scratch memory) and about 220 scalar ones kept in lanes of them; with heads
// of 64 168 (fp16 one more) and 220 to 240.
constexpr int kKeyCost = 20, kRowCost = 30, kItemCost = 80;  // a step of keys, of rows; a tile
constexpr int kLeast = 160;                                  // a share

struct Back {
    float *rows;    // [n_heads][2 blocks][4][32]
    float *norms;   // fp16: the largest |do| of a block's rows [n_heads][blocks], |v| [n_kv][blocks], |D| [n_heads][blocks]
    int4 *tab;      // a tile's keys [x, y) and rows [z, w): what its rows see, what sees its keys
    int64_t *line;  // [2 tiles + 1]: where the tiles of keys begin, then those of rows (of all heads)
    int *inside;    // [n_kv * groups]: the tile (of all heads) that a share begins inside of, or -1
    float *part;    // [n_kv * groups][2][arrays][4 waves][32 D]
    int blocks;
    int tiles;      // of 128
    int groups;     // shares of a key/value head, at most; 0: tiles
};

struct Line {
    int64_t total;
    int groups;
    __device__ __forceinline__ void set(const Back &b) {
        total = uniform64(b.line[2 * b.tiles]);
        const int64_t n = total / kLeast;
        groups = n < 1 ? 1 : n < b.groups ? static_cast<int>(n) : b.groups;
    }
    // share g's first place: a quotient by way of 64-bit floats, then put right (a division of 64-bit
    // whole numbers is a hundred instructions)
    __device__ __forceinline__ int64_t begin(int g) const { return quotient(total * g, groups); }
    __device__ __forceinline__ static int64_t quotient(int64_t a, int64_t b) {
        int64_t q = static_cast<int64_t>(static_cast<double>(a) / static_cast<double>(b));
        if (q * b > a) --q;
        else if ((q + 1) * b <= a) ++q;
        return uniform64(q);
    }
};

// Steps of `cost` that begin in the share [s0, s1), of n (a tile without any counts as one) of a tile
// that begins at c.
__device__ __forceinline__ int2 steps_in(int64_t s0, int64_t s1, int64_t c, int n, int cost) {
    const int64_t m = n < 1 ? 1 : n;
    const int64_t x = s0 > c ? (s0 - c + cost - 1) / cost : 0, y = s1 > c ? (s1 - c + cost - 1) / cost : 0;
    return make_int2(static_cast<int>(x < m ? x : m), static_cast<int>(y < m ? y : m));
}

// Steps of `unit` positions over [x, y), whole ones.
__device__ __forceinline__ int steps_over(int x, int y, int unit) { return x < y ? (y - 1) / unit - x / unit + 1 : 0; }

// A lane's own search in offsets `cu` (in LDS or not): the rows of row t's sequence, or [t, t).
template <typename Offsets>
__device__ __forceinline__ int2 sequence_of_lane(const Attn &a, Offsets cu, int t) {
    int lo = 0, hi = a.batch + 1;  // the first offset past t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    if (lo == 0 || lo > a.batch) return make_int2(t, t);
    const int s = cu[lo - 1], e = cu[lo];
    return make_int2(s < 0 ? 0 : s, e > a.tokens ? a.tokens : e);
}

// The table and the line, by one workgroup: a tile a thread, 256 at a time.  It is the latency of what it waits for
// that counts: the offsets come to LDS at once where they fit, and what a thread has found stays with it.
__device__ __forceinline__ void make_line(const Attn &a, const Back &b) {
    constexpr int LDS_OFFSETS = 1024;
    __shared__ int64_t sum[2][4];
    __shared__ int offsets[LDS_OFFSETS];
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
    const bool fit = a.cu && a.batch < LDS_OFFSETS;
    if (fit) {
#pragma unroll
        for (int x = 0; x < LDS_OFFSETS; x += 256)
            if (x + static_cast<int>(threadIdx.x) <= a.batch) offsets[x + threadIdx.x] = a.cu[x + threadIdx.x];
        __syncthreads();
    }
    const int begin = !a.cu ? 0 : fit ? offsets[0] : a.cu[0], end = !a.cu ? a.tokens : fit ? offsets[a.batch] : a.cu[a.batch];
    auto sequence = [&](int t) {
        return !a.cu ? make_int2(0, a.tokens) : fit ? sequence_of_lane(a, offsets, t) : sequence_of_lane(a, a.cu, t);
    };
    int64_t at[2] = {0, 0}, of_rows = 0;  // (rows' tiles begin behind all keys')
#pragma unroll 1
    for (int t0 = 0; t0 < b.tiles; t0 += 256) {
        const int t = t0 + threadIdx.x;
        int64_t cost[2] = {0, 0}, upto[2];
        if (t < b.tiles) {
            const int first = t * kOwn > begin ? t * kOwn : begin;
            int last = t * kOwn + kOwn < a.tokens ? t * kOwn + kOwn - 1 : a.tokens - 1;
            last = last < end ? last : end - 1;
            int4 r = make_int4(0, 0, 0, 0);
            if (first <= last) {
                const int2 x = sequence(first), y = sequence(last);
                r.x = a.window && first - a.window + 1 > x.x ? first - a.window + 1 : x.x;
                r.y = last + 1;
                r.z = first;
                r.w = a.window && last + a.window < y.y ? last + a.window : y.y;
            }
            b.tab[t] = r;
            cost[0] = static_cast<int64_t>(steps_over(r.z, r.w, kRows)) * a.group * kKeyCost + kItemCost;
            cost[1] = static_cast<int64_t>(steps_over(r.x, r.y, kTile) * kRowCost + kItemCost) * a.group;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            upto[k] = cost[k];
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int64_t x = __shfl_up(upto[k], o);
                if (l >= o) upto[k] += x;
            }
            if (l == 63) sum[k][w] = upto[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            for (int i = 0; i < w; ++i) upto[k] += sum[k][i];
            upto[k] += at[k] - cost[k];
            at[k] += sum[k][0] + sum[k][1] + sum[k][2] + sum[k][3];
        }
        if (t < b.tiles) {
            b.line[t] = upto[0];
            of_rows = upto[1];
            if (b.tiles > 256) b.line[b.tiles + t] = of_rows;
        }
        __syncthreads();
    }
    for (int t = threadIdx.x; t < b.tiles; t += 256) {
        if (b.tiles > 256) of_rows = b.line[b.tiles + t];
        b.line[b.tiles + t] = at[0] + of_rows;
    }
    if (threadIdx.x == 0) b.line[2 * b.tiles] = at[0] + at[1];
}

// One workgroup per 64 rows and head; heads from n_heads on are those of v, the last makes the line.
template <int DT, int D>
__global__ __launch_bounds__(256) void attn_rows_kernel(const Attn a, const Back b) {
    constexpr int CH = D / 8, RPP = 256 / CH;
    __shared__ float most[2][4];
    const int head = blockIdx.y, ch = threadIdx.x % CH;
    if (head == static_cast<int>(gridDim.y) - 1) {
        if (blockIdx.x == 0) make_line(a, b);
        return;
    }
    const bool of_v = head >= a.n_heads;
    float worst = 0.f, worst_d = 0.f;
    constexpr int N = kTile / RPP;
    u32x4_t go[N], out[N];
    float2 stats[N];
#pragma unroll
    for (int x = 0; x < N; ++x) {  // (all are asked for at once; rows that are not there: the last one)
        int r = blockIdx.x * kTile + x * RPP + threadIdx.x / CH;
        r = r < a.tokens ? r : a.tokens - 1;
        stats[x] = a.stats[static_cast<int64_t>(r) * a.n_heads + (of_v ? 0 : head)];
        go[x] = *reinterpret_cast<const u32x4_t *>((of_v ? a.v.at(r, head - a.n_heads) : a.dout.at(r, head)) + ch * 8);
        out[x] = go[x];
        if (!of_v) out[x] = *reinterpret_cast<const u32x4_t *>(a.o.at(r, head) + ch * 8);
    }
#pragma unroll
    for (int x = 0; x < N; ++x) {
        const int i = x * RPP + threadIdx.x / CH, r = blockIdx.x * kTile + i;
        float2 ml = r < a.tokens ? stats[x] : make_float2(0.f, 0.f);
        float f[8], o[8], d = 0.f, sq = 0.f;
        unpack8<DT>(go[x], f);
        unpack8<DT>(out[x], o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sq = fmaf(f[e], f[e], sq);
            d = fmaf(f[e], o[e], d);
        }
#pragma unroll
        for (int o = 1; o < CH; o <<= 1) {
            d += __shfl_xor(d, o);
            sq += __shfl_xor(sq, o);
        }
        const bool none = ml.y == 0.f;  // a row of no sequence, whatever lies there
        if (!none && sq < INFINITY) worst = fmaxf(worst, sq);  // (what sees an odd one is NaN)
        if (of_v || ch) continue;
        if (none) d = 0.f;
        else if (!(fabsf(d) < INFINITY && fabsf(ml.x) < INFINITY)) ml = make_float2(NAN, NAN);  // (an odd do or out: an odd d)
        else worst_d = fmaxf(worst_d, fabsf(d));
        const float ll = (ml.y == 0.f ? 0.f : log2f(ml.y)) - kTop<DT>;
        float *p = b.rows + (static_cast<int64_t>(head) * b.blocks + blockIdx.x) * 256 + (i >> 5) * 128 + (i & 31);
        p[0] = ml.x;
        p[32] = ll;
        p[64] = ml.x + ll;
        p[96] = -d;
    }
    if constexpr (DT == NF4_F16) {
        worst = wave_max(worst);
        worst_d = wave_max(worst_d);
        if ((threadIdx.x & 63) == 0) {
            most[0][threadIdx.x >> 6] = worst;
            most[1][threadIdx.x >> 6] = worst_d;
        }
        __syncthreads();
        if (threadIdx.x < 2 && !(of_v && threadIdx.x)) {
            const float *m = most[threadIdx.x];
            const float x = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            b.norms[static_cast<int64_t>(head + (threadIdx.x ? a.n_heads + a.n_kv : 0)) * b.blocks + blockIdx.x] = threadIdx.x ? x : sqrtf(x);
        }
    }
}

// fp16's dS, of at most `bound` = |do| |v| + |D|, are multiplied by this power of two (beside the 2^15 of P),
// so that the largest is near 2^15; a plain fp16 of them would be 0 for the gradients of a loss that is not
// scaled.  (D by itself: it has the v of every key that the row sees in it, which can be far larger than
// those at hand.)
__device__ __forceinline__ float ds_scale(float bound) {
    int e = 0;
    bound *= 1.01f;
    if (bound > 0.f && bound < INFINITY) (void)frexpf(bound, &e);
    return ldexpf(1.f, -e);
}

// The largest of n numbers of `heads` heads each, `blocks` apart, and of those `other` behind them: of both at a
// time, since it is the loads' latency that counts.
__device__ __forceinline__ float2 most_of(const float *p, int n, int heads, int64_t blocks, int64_t other) {
    float2 v = make_float2(0.f, 0.f);
    for (int h = 0; h < heads; ++h, p += blocks)
        for (int i = thread_here() & 63; i < n; i += 64) {
            const float x = p[i], y = p[i + other];
            v.x = fmaxf(v.x, x);
            v.y = fmaxf(v.y, y);
        }
    return make_float2(wave_max(v.x), wave_max(v.y));
}

// |x|^2 of a lane's row, from its operands
template <int DT, int D>
__device__ __forceinline__ float square_of(const u32x4_t (&f)[D / 16]) {
    float s = 0.f;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
        float v[8];
        unpack8<DT>(f[x], v);
#pragma unroll
        for (int i = 0; i < 8; ++i) s = fmaf(v[i], v[i], s);
    }
    return s + other_half(s);
}

// A tile of rows: keys [x, y) are seen, steps [u.x, u.y) are this share's; `part` where they are not all.
template <int DT, int D>
__device__ __forceinline__ void dq_body(const Attn &a, const Back &b, int head, int tile, int2 keys, int2 u,
                                        float *part, uint8_t *lds) {
    constexpr int KS = D / 16, DN = D / 32, TB = kTileBytes<D>;
    const int tid = thread_here(), w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63;
    const int n = l & 31, kvh = head / a.group;
    const int r = tile * kOwn + w * 32 + n;
    const int first = (keys.x & ~(kTile - 1)) + u.x * kTile;
    int last = (keys.x & ~(kTile - 1)) + u.y * kTile;
    last = last < keys.y ? last : keys.y;

    u32x4_t q[KS], go[KS];
    own_operand<D>(q, a.q.at(r, head), r < a.tokens, l);
    own_operand<D>(go, a.dout.at(r, head), r < a.tokens, l);
    const float *rows = b.rows + (static_cast<int64_t>(head) * b.blocks * 2 + (r < a.tokens ? r >> 5 : 0)) * 128 + (r & 31);
    const float m = rows[0], ll = rows[32], base = rows[64], delta = rows[96];
    Stager<D, kTile> sk, sv;
    sk.set(a.k, kvh, first, tid);
    sv.set(a.v, kvh, first, tid);
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) uint8_t *)lds));
    const uint32_t mine = __builtin_amdgcn_readfirstlane(lds0 + w * 1024);
    int k = u.x < u.y ? first : last, st = 0;
    if (k < last) {
        const int skip = keys.x > k ? keys.x - k : 0;  // (as in the forward pass)
        sk.send(mine, last - k, skip);
        sv.send(mine + 2 * TB, last - k, skip);
    }
    // (what the rows see is found while all that is on its way)
    const int2 seen = keys_of(a, r);
    Span sp;
    sp.set(seen);
    const bool near = __all(!(seen.x < seen.y) || fabsf(m) < kNear);
    float fs = 1.f;
    if constexpr (DT == NF4_F16) {
        const int b0 = first >> 6, nb = u.y - u.x;
        fs = ds_scale(sqrtf(square_of<DT, D>(go)) * most_of(b.norms + static_cast<int64_t>(a.n_heads + kvh) * b.blocks + b0, nb, 1, 0, 0).x + fabsf(delta));
    }
    // (the probabilities are used for dS only: their scale goes into the exponent)
    const float mul = near ? a.c : 1.f, sub = (near ? base : 0.f) - log2f(fs);
    const uint32_t ra = lds0 + row_address<D>(l), ca = lds0 + channel_address<D>(l);

    float16_t acc[DN];
#pragma unroll
    for (int x = 0; x < DN; ++x) acc[x] = (float16_t){};
#pragma unroll 1
    for (; k < last; k += kTile, st ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (k + kTile < last) {
            sk.send(mine + (st ^ 1) * TB, last - k - kTile);
            sv.send(mine + (2 + (st ^ 1)) * TB, last - k - kTile);
        }
        const uint32_t ka = ra + st * TB, va = ra + (2 + st) * TB, kt = ca + st * TB;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (sp.none(k + 32 * h, 32)) continue;
            constexpr int AHEAD = D == 128 ? 4 : 2;  // steps of k's and v's operands under way
            u32x4_t kf[AHEAD], vf[AHEAD];
#pragma unroll
            for (int x = 0; x < AHEAD; ++x) {
                kf[x] = rows_operand<D>(ka, h, x);
                vf[x] = rows_operand<D>(va, h, x);
            }
            float16_t sc = (float16_t){}, dp;
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] = delta;
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int x = 0; x < KS; ++x) {
                sc = mfma32<DT>(kf[x % AHEAD], q[x], sc);
                dp = mfma32<DT>(vf[x % AHEAD], go[x], dp);
                if (x + AHEAD < KS) {
                    kf[x % AHEAD] = rows_operand<D>(ka, h, x + AHEAD);
                    vf[x % AHEAD] = rows_operand<D>(va, h, x + AHEAD);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            u32x4_t tf[2][DN];
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int d = 0; d < DN; ++d) tf[x][d] = channels_operand<D>(kt, 2 * h + x, d);
            __builtin_amdgcn_sched_barrier(0);
            if (__builtin_expect(!near, 0)) {
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = capped(exponent(sc[e], a.c, m) - ll, kTop<DT>);
            }
            if (!sp.full(k + 32 * h, 32)) {
                const uint64_t see = seen_bits(seen, k);
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (!bit_of(see, h, e)) {
                        sc[e] = a.c < 0.f && near ? INFINITY : -INFINITY;
                        dp[e] = 0.f;  // (a NaN of v that the row does not see)
                    }
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) sc[e] = __builtin_amdgcn_exp2f(fmaf(sc[e], mul, -sub)) * dp[e];
            const u32x4_t pf[2] = {operand_of<DT>(sc, 0), operand_of<DT>(sc, 1)};
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int d = 0; d < DN; ++d) acc[d] = mfma32<DT>(tf[x][d], pf[x], acc[d]);
            __builtin_amdgcn_s_setprio(0);
        }
    }
    const int2 own = make_int2(seen.x > first ? seen.x : first, seen.y < last ? seen.y : last);  // of this share
    const bool some = own.x < own.y;
    if (part) part += w * 32 * D;
    const bool nan = some && base != base;
    uint32_t again = rows_where(some && !nan && any_nan(acc));
    if (again) {  // but for what an infinity of k explains
        uint32_t by[D / 64];
        nan_by<DT, D, true>(a.k, kvh, sp.lo > first ? sp.lo : first, sp.hi < last ? sp.hi : last, own, by);
        again &= rows_where(unexplained<D>(acc, by));
    }
    if (!some) fill_of(acc, 0.f);
    else if (nan) fill_of(acc, NAN);
    const float f = a.scale * (ldexpf(1.f, -static_cast<int>(kTop<DT>)) / fs);
    if (part) {
#pragma unroll
        for (int x = 0; x < DN; ++x) acc[x] *= f;
        store_part<D>(part, acc);
    } else if (r < a.tokens && !(again >> n & 1)) {
        store_own<DT, D>(a.dq.to(r, head), acc, f);
    }
    if (!again) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (as in the forward pass)
#pragma unroll 1
    for (uint32_t left = again; left; left &= left - 1) {
        const int i = __builtin_ctz(left), row = tile * kOwn + w * 32 + i;
        float o[D / 64];
        row_backward<DT, D>(a, head, row, __builtin_amdgcn_readlane(own.x, i), __builtin_amdgcn_readlane(own.y, i), o);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) o[x] *= a.scale;
        if (part) store_part_row<D>(part, i, o);
        else store_row<DT, D>(a.dq.to(row, head), o);
    }
}

// The keys' workgroup holds its k and its sums in registers (160 of the 256 that two waves a SIMD leave)
// and its v in LDS: with v in registers too, the operands of each product were waited for one at a time
// (8192 tokens of 28 heads, the whole backward pass: a third longer), and tiles are of 32 rows, so that two
// workgroups' LDS fits a CU.
template <int D>
constexpr int kKeyLds = kOwn * D * 2 + 4 * kRows * D * 2 + 2 * 1024;  // v; q and do, two stages; their rows' numbers
template <int D>
constexpr int kBackLds = (kKeyLds<D> > 4 * kTileBytes<D> ? kKeyLds<D> : 4 * kTileBytes<D>) + 64;

// A tile of keys: rows [x, y) see them, steps [u.x, u.y) are this share's; `part` where they are not all.
template <int DT, int D>
__device__ __forceinline__ void dkv_body(const Attn &a, const Back &b, int kvh, int tile, int2 rows, int2 units,
                                         float *part, uint8_t *lds) {
    constexpr int KS = D / 16, DN = D / 32, RB = kRows * D * 2, VB = kOwn * D * 2;
    const int tid = thread_here(), w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63;
    const int g = l >> 5, n = l & 31;
    const int j = tile * kOwn + w * 32 + n;
    const int t0 = rows.x / kRows, per = steps_over(rows.x, rows.y, kRows);

    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) uint8_t *)lds));
    const uint32_t mine = __builtin_amdgcn_readfirstlane(lds0 + w * 1024);
    const uint32_t tiles0 = mine + VB, rows0 = __builtin_amdgcn_readfirstlane(lds0 + VB + 4 * RB);
    Stager<D, kOwn> sv;
    Stager<D, kRows> sq, sg;
    sv.set(a.v, kvh, tile * kOwn, tid);
    if (units.x < units.y) sv.send(mine, a.tokens - tile * kOwn);
    u32x4_t kf[KS];
    own_operand<D>(kf, a.k.at(j, kvh), j < a.tokens, l);
    // unit (head of the group, tile of rows), the next one
    int uh = per ? units.x / per : 0, ut = units.x - uh * per;
    sq.set(a.q, kvh * a.group + uh, (t0 + ut) * kRows, tid);
    sg.set(a.dout, kvh * a.group + uh, (t0 + ut) * kRows, tid);
    int t = ut, st = 0;
    auto numbers = [&](int h) {  // of the rows of tile t0 of a head
        return b.rows + (static_cast<int64_t>(kvh * a.group + h) * b.blocks * 2 + t0) * 128;
    };
    const float *rw_next = numbers(uh) + ut * 128;
    auto send = [&](int st) {
        const int left = rows.y - (t0 + ut) * kRows, skip = ut ? 0 : rows.x - t0 * kRows;
        sq.send(tiles0 + st * RB, left, skip);
        sg.send(tiles0 + (2 + st) * RB, left, skip);
        if (w == 0)  // (512 bytes: the upper lanes' are past the end, zeros)
            lds_dma16(rows0 + st * 1024, l * 16, make_rsrc(reinterpret_cast<const float *>(uniform64(reinterpret_cast<int64_t>(rw_next))), 512), 0);
        rw_next += 128;
        if (++ut == per) {
            ut = 0;
            ++uh;
            sq.begin(a.q, kvh * a.group + uh, t0 * kRows);
            sg.begin(a.dout, kvh * a.group + uh, t0 * kRows);
            rw_next = numbers(uh);
        }
    };
    const uint32_t va = lds0 + w * 32 * D * 2 + row_address<D>(l);
    const uint32_t ra = lds0 + VB + row_address<D>(l), ca = lds0 + VB + channel_address<D>(l);
    if (units.x < units.y) send(0);
    // (what sees the keys is found while all that is on its way)
    const int2 seen = rows_of(a, j);
    Span sp;
    sp.set(seen);
    float fs = 1.f;
    if constexpr (DT == NF4_F16) {
        u32x4_t vf[KS];
        own_operand<D>(vf, a.v.at(j, kvh), j < a.tokens, l);
        const int b0 = t0 * kRows / kTile, nb = per ? (rows.y - 1) / kTile - b0 + 1 : 0;
        const float2 most = most_of(b.norms + static_cast<int64_t>(kvh * a.group) * b.blocks + b0, nb, a.group, b.blocks,
                                    static_cast<int64_t>(a.n_heads + a.n_kv) * b.blocks);
        fs = ds_scale(sqrtf(square_of<DT, D>(vf)) * most.x + most.y);
    }
    float16_t dk[DN], dv[DN];
#pragma unroll
    for (int x = 0; x < DN; ++x) dk[x] = dv[x] = (float16_t){};
#pragma unroll 1
    for (int u = units.x; u < units.y; ++u, st ^= 1) {
        const int r = (t0 + t) * kRows;
        if (++t == per) t = 0;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (u + 1 < units.y) send(st ^ 1);
        if (sp.none(r, kRows)) continue;
        const uint32_t qa = ra + st * RB, ga = ra + (2 + st) * RB, rw = rows0 + st * 1024 + g * 16;
        auto row4 = [&](int kind, int e) {  // rows 2 e + 4 g .. of a kind
            return __builtin_bit_cast(float4_t, lds16(rw + kind * 128 + e * 8));
        };
        constexpr int AHEAD = 2;  // steps of the operands of q, do and v under way
        u32x4_t qf[AHEAD], gf[AHEAD], vf[AHEAD];
        auto read = [&](int x) {
            qf[x % AHEAD] = rows_operand<D>(qa, 0, x);
            gf[x % AHEAD] = rows_operand<D>(ga, 0, x);
            vf[x % AHEAD] = rows_operand<D>(va, 0, x);
        };
#pragma unroll
        for (int x = 0; x < AHEAD; ++x) read(x);
        float16_t sc = (float16_t){}, dp;
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const float4_t d = row4(3, e);
#pragma unroll
            for (int i = 0; i < 4; ++i) dp[e + i] = d[i];
        }
        const float row_m = *reinterpret_cast<const __attribute__((address_space(3))) float *>(static_cast<uintptr_t>(rw - g * 16 + n * 4));
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int x = 0; x < KS; ++x) {
            sc = mfma32<DT>(qf[x % AHEAD], kf[x], sc);
            dp = mfma32<DT>(gf[x % AHEAD], vf[x % AHEAD], dp);
            if (x + AHEAD < KS) read(x + AHEAD);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        const bool near = __all(fabsf(row_m) < kNear);
        u32x4_t tf[2][DN];
        auto read_t = [&](int i) {  // operands of the last products' i-th quarter: do and q in turn
#pragma unroll
            for (int d = 0; d < DN; ++d)
                tf[i & 1][d] = channels_operand<D>(ca + ((i & 1 ? 0 : 2) + st) * RB, i >> 1, d);
        };
        if (__builtin_expect(near, 1)) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const float4_t base = row4(2, e);
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[e + i] = fmaf(sc[e + i], a.c, -base[i]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const float4_t m = row4(0, e), ll = row4(1, e);
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[e + i] = capped(exponent(sc[e + i], a.c, m[i]) - ll[i], kTop<DT>);
            }
        }
        if (!sp.full(r, kRows)) {
            const uint64_t see = seen_bits(seen, r);
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (!bit_of(see, 0, e)) {
                    sc[e] = -INFINITY;
                    dp[e] = 0.f;  // (a row's NaN that the key is not seen by)
                }
        }
        read_t(0);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sc[e] = __builtin_amdgcn_exp2f(sc[e]);
            dp[e] *= sc[e];
            if constexpr (DT == NF4_F16) dp[e] *= fs;
        }
        const u32x4_t pf[4] = {operand_of<DT>(sc, 0), operand_of<DT>(dp, 0), operand_of<DT>(sc, 1), operand_of<DT>(dp, 1)};
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i < 3) read_t(i + 1);
#pragma unroll
            for (int d = 0; d < DN; ++d) {
                if (i & 1) dk[d] = mfma32<DT>(tf[1][d], pf[i], dk[d]);
                else dv[d] = mfma32<DT>(tf[0][d], pf[i], dv[d]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    const bool some = seen.x < seen.y;
    if (part) part += w * 32 * D;
    uint32_t again = rows_where(some && (any_nan(dk) || any_nan(dv)));
    if (!some) {
        fill_of(dk, 0.f);
        fill_of(dv, 0.f);
    }
    // rows of this share's heads [x0, x1), the last head first
    int h = per ? (units.y - 1) / per : -1;
    auto span = [&](int &x0, int &x1) {
        x0 = (t0 + (units.x > h * per ? units.x - h * per : 0)) * kRows;
        x1 = (t0 + (units.y < (h + 1) * per ? units.y - h * per : per)) * kRows;
    };
    if (again) {
        // a key that sees a row whose numbers are NaN has NaN: the last rows first, which most keys see
        bool nan = false;
#pragma unroll 1
        for (; h >= 0 && h * per + per > units.x && (again & ~rows_where(nan)); --h) {
            int x0, x1;
            span(x0, x1);
            for (int x = x1 - 64; x > x0 - 64 && (again & ~rows_where(nan)); x -= 64) {
                const int row = x + l;
                float base = 0.f;
                if (row >= x0) base = numbers(h)[(row / kRows - t0) * 128 + 64 + row % kRows];
                nan |= (__ballot(base != base) & below(seen.y - x) & ~below(seen.x - x)) != 0;
            }
        }
        nan = nan && some;
        if (nan) {
            fill_of(dk, NAN);
            fill_of(dv, NAN);
        }
        again &= ~rows_where(nan);
    }
    const float one = ldexpf(1.f, -static_cast<int>(kTop<DT>)), f = a.scale * (one / fs);
    if (part) {
#pragma unroll
        for (int x = 0; x < DN; ++x) {
            dk[x] *= f;
            dv[x] *= one;
        }
        store_part<D>(part, dk);
        store_part<D>(part + kOwn * D, dv);
    } else if (j < a.tokens && !(again >> n & 1)) {
        store_own<DT, D>(a.dk.to(j, kvh), dk, f);
        store_own<DT, D>(a.dv.to(j, kvh), dv, one);
    }
    if (!again) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (as in the forward pass)
#pragma unroll 1
    for (uint32_t left = again; left; left &= left - 1) {
        const int i = __builtin_ctz(left), key = tile * kOwn + w * 32 + i;
        const int r0 = __builtin_amdgcn_readlane(seen.x, i), r1 = __builtin_amdgcn_readlane(seen.y, i);
        float gk[D / 64] = {}, gv[D / 64] = {};
        for (h = units.x / per; h * per < units.y; ++h) {
            int x0, x1;
            span(x0, x1);
            key_backward<DT, D>(a, kvh * a.group + h, key, r0 > x0 ? r0 : x0, r1 < x1 ? r1 : x1, gk, gv);
        }
#pragma unroll
        for (int x = 0; x < D / 64; ++x) gk[x] *= a.scale;
        if (part) {
            store_part_row<D>(part, i, gk);
            store_part_row<D>(part + kOwn * D, i, gv);
        } else {
            store_row<DT, D>(a.dk.to(key, kvh), gk);
            store_row<DT, D>(a.dv.to(key, kvh), gv);
        }
    }
}

// A share's slot of parts: 0 of the tile that it begins inside of, 1 of the one that it begins.
template <int D>
__device__ __forceinline__ float *slot_of(const Back &b, int kvh, int g, int i) {
    return b.part + ((static_cast<int64_t>(kvh) * b.groups + g) * 2 + i) * 2 * kOwn * D;
}

template <int DT, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void attn_bwd_kernel(const Attn a, const Back b) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBackLds<D>];
    __shared__ int cursor[2];  // shares: the next tile of the line and head of the group
    if (b.groups) {
        const int g = blockIdx.x / a.n_kv, kvh0 = blockIdx.x % a.n_kv, l = threadIdx.x & 63;
        Line line;
        line.set(b);
        int *inside = b.inside + kvh0 * b.groups + g;
        if (threadIdx.x == 0) *inside = -1;
        if (g >= line.groups) return;
        const int64_t s0 = line.begin(g);
        // the last tile (of all heads) that begins at or before the share
        int e = 0;
        for (int n = 2 * b.tiles; n > 1;) {
            const int step = (n + 63) >> 6, i = l * step;
            const int c = __popcll(__ballot(i < n && b.line[e + i] <= s0));  // (at least 1)
            e += (c - 1) * step;
            n = n - (c - 1) * step < step ? n - (c - 1) * step : step;
        }
        if (threadIdx.x == 0) {
            int h = 0;
            if (e >= b.tiles) {
                const int4 r = b.tab[e - b.tiles];
                h = static_cast<int>((s0 - b.line[e]) / (steps_over(r.x, r.y, kTile) * kRowCost + kItemCost));
            }
            cursor[0] = e;
            cursor[1] = h;
        }
    }
    // (what a tile needs to know is read again for each: kept over the tiles' work, it took registers that
    // their loops spilled)
    for (;;) {
        __syncthreads();  // the cursor is there, and the tile before is read
        int kvh = blockIdx.x % a.n_kv, e, h;
        if (b.groups) {
            e = __builtin_amdgcn_readfirstlane(cursor[0]);
            h = __builtin_amdgcn_readfirstlane(cursor[1]);
            if (e >= 2 * b.tiles) return;
        } else {
            const int i = blockIdx.x / a.n_kv - b.tiles;
            e = i < 0 ? i + b.tiles : 2 * b.tiles - 1 - i / a.group;  // (the last rows see most: first)
            h = i < 0 ? 0 : i % a.group;
        }
        const bool of_keys = e < b.tiles;
        const int tile = of_keys ? e : e - b.tiles;
        const int4 r = b.tab[tile];
        const int x = __builtin_amdgcn_readfirstlane(of_keys ? r.z : r.x), y = __builtin_amdgcn_readfirstlane(of_keys ? r.w : r.y);
        const int n = of_keys ? steps_over(x, y, kRows) * a.group : steps_over(x, y, kTile);
        int2 u = make_int2(0, n);
        float *part = nullptr;
        if (b.groups) {
            const int g = blockIdx.x / a.n_kv, cost = of_keys ? kKeyCost : kRowCost;
            Line line;
            line.set(b);
            const int64_t c = uniform64(b.line[e]) + static_cast<int64_t>(h) * (n * cost + kItemCost);
            const int64_t s1 = line.begin(g + 1);
            if (c >= s1) return;
            u = steps_in(line.begin(g), s1, c, n, cost);
            u.x = __builtin_amdgcn_readfirstlane(u.x);
            u.y = __builtin_amdgcn_readfirstlane(u.y);
            __syncthreads();
            if (threadIdx.x == 0) {
                const bool on = of_keys || h + 1 == a.group;
                cursor[0] = on ? e + 1 : e;
                cursor[1] = on ? 0 : h + 1;
            }
            if (u.x >= u.y) continue;
            if (u.x > 0 && threadIdx.x == 0)
                b.inside[kvh * b.groups + g] = of_keys ? tile : b.tiles + tile * a.group + h;
            if (u.x > 0 || u.y < n) part = slot_of<D>(b, kvh, g, u.x == 0);
            if (n == 0) u.y = 0;
        }
        if (of_keys) dkv_body<DT, D>(a, b, kvh, tile, make_int2(x, y), u, part, lds);
        else dq_body<DT, D>(a, b, kvh * a.group + h, tile, make_int2(x, y), u, part, lds);
        if (!b.groups) return;
    }
}

// The tile that a share begins inside of, where it is the first one to: 32 of its rows (or keys) a
// workgroup, whose parts are summed in the shares' order.  Grid x = rows / 32 of dq or dk, then of dv,
// y = shares of all heads.
template <int DT, int D>
__global__ __launch_bounds__(256) void attn_bwd_join_kernel(const Attn a, const Back b) {
    __shared__ __attribute__((aligned(16))) uint16_t lds[32 * (D + 8)];
    const int kvh = blockIdx.y / b.groups, w = blockIdx.x & 3, array = blockIdx.x >> 2;
    int g = blockIdx.y % b.groups;
    const int *inside = b.inside + kvh * b.groups;
    const int i = g - 1 + (threadIdx.x & 63);  // the share before, this one and those behind it
    const int near = i >= 0 && i < b.groups ? inside[i] : -1;
    const int e = __builtin_amdgcn_readlane(near, 1);
    if (e < 0 || (array && e >= b.tiles) || __builtin_amdgcn_readlane(near, 0) == e) return;
    int end = g + __builtin_ctzll(~(__ballot(near == e) >> 1));  // the first share that is not inside of it
    if (end == g + 63)
        while (end < b.groups && inside[end] == e) ++end;
    const int at = (array * kOwn + w * 32) * D + threadIdx.x * 4;
    float4_t v[D / 32];
    const float *part = slot_of<D>(b, kvh, g - 1, 1) + at;
#pragma unroll
    for (int x = 0; x < D / 32; ++x) v[x] = *reinterpret_cast<const float4_t *>(part + x * 1024);
    part = slot_of<D>(b, kvh, g, 0) + at;
    constexpr int64_t NEXT = 4 * kOwn * D;  // the next share's slot 0
    constexpr int BATCH = 4;                // parts whose loads are under way: it is their latency that counts
    for (; g < end; g += BATCH, part += BATCH * NEXT) {
        float4_t f[BATCH][D / 32];
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
#pragma unroll
            for (int x = 0; x < D / 32; ++x) {
                f[i][x] = (float4_t){0.f, 0.f, 0.f, 0.f};
                if (g + i < end) f[i][x] = *reinterpret_cast<const float4_t *>(part + i * NEXT + x * 1024);
            }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
#pragma unroll
            for (int x = 0; x < D / 32; ++x) v[x] += f[i][x];
    }
    const bool of_keys = e < b.tiles;
    const int tile = of_keys ? e : (e - b.tiles) / a.group, head = of_keys ? kvh : kvh * a.group + (e - b.tiles) % a.group;
#pragma unroll
    for (int x = 0; x < D / 32; ++x) join_put<DT, D>(lds, x * 256 + threadIdx.x, v[x]);
    join_write<D>(!of_keys ? a.dq : array ? a.dv : a.dk, head, tile * kOwn + w * 32, a.tokens, lds);
}

// ------------------------------------------------------------------------- host

// Strides of a dimension of one do not count.
int take(Strided &s, const void *p, int64_t tok, int64_t head, int64_t tokens, int heads) {
    s.p = static_cast<const uint16_t *>(p);
    s.tok = tokens > 1 ? tok : 0;
    s.head = heads > 1 ? head : 0;
    if (!p || s.tok < 0 || s.head < 0) return NF4_ERR_ARG;
    if (!aligned(p, 16) || s.tok % 8 || s.head % 8 || s.tok > (1 << 23)) return NF4_ERR_UNSUPPORTED;
    return NF4_OK;
}

// A gradient, whose rows must be apart.
int take(Strided &s, const nf4_grad *g, int64_t tokens, int heads, int head_dim) {
    if (!g) return NF4_ERR_ARG;
    const int st = take(s, g->p, g->tok, g->head, tokens, heads);
    if (st != NF4_OK) return st;
    const int64_t row = (heads - 1) * s.head + head_dim, col = (tokens - 1) * s.tok + head_dim;
    const bool by_tok = (tokens == 1 || s.tok >= row) && (heads == 1 || s.head >= head_dim);
    const bool by_head = (heads == 1 || s.head >= col) && (tokens == 1 || s.tok >= head_dim);
    return by_tok || by_head ? NF4_OK : NF4_ERR_ARG;
}

int fill(Attn &a, const nf4_attn *in) {
    if (!in) return NF4_ERR_ARG;
    if (in->dtype != NF4_F16 && in->dtype != NF4_BF16) return NF4_ERR_ARG;
    if (in->tokens < 0 || in->window < 0 || in->max_len < 0 || in->batch < 0) return NF4_ERR_ARG;
    if (in->n_heads < 1 || in->n_kv < 1 || in->n_heads % in->n_kv) return NF4_ERR_ARG;
    if (in->head_dim != 64 && in->head_dim != 128) return NF4_ERR_UNSUPPORTED;
    const float c = fabsf(in->scale) * kLog2e;
    if (!(c < INFINITY)) return NF4_ERR_ARG;  // NaN too
    if (!in->cu && in->batch != 1 && in->tokens) return NF4_ERR_ARG;
    if (in->tokens > (1 << 23) || in->n_heads > 1024 || in->batch > (1 << 20) ||
        in->tokens * in->n_heads > (1 << 30))
        return NF4_ERR_UNSUPPORTED;
    if (in->tokens == 0) return NF4_OK;
    if (!aligned(in->cu, 4)) return NF4_ERR_UNSUPPORTED;
    int st = take(a.q, in->q, in->q_tok, in->q_head, in->tokens, in->n_heads);
    if (st == NF4_OK) st = take(a.k, in->k, in->k_tok, in->k_head, in->tokens, in->n_kv);
    if (st == NF4_OK) st = take(a.v, in->v, in->v_tok, in->v_head, in->tokens, in->n_kv);
    if (st != NF4_OK) return st;
    a.cu = in->cu;
    a.batch = in->batch;
    a.tokens = static_cast<int>(in->tokens);
    a.window = static_cast<int>(in->window < in->tokens ? in->window : 0);
    a.n_heads = in->n_heads;
    a.n_kv = in->n_kv;
    a.group = in->n_heads / in->n_kv;
    a.c = copysignf(fmaxf(c, 1.2e-38f), in->scale);  // (a normal number's least)
    a.scale = in->scale;
    return NF4_OK;
}

int tiles_of(const nf4_attn *in, int n) { return static_cast<int>((in->tokens + n - 1) / n); }

template <int DT, int D>
int forward(const Attn &a, const Pieces &pc, int tiles, hipStream_t s) {
    hipLaunchKernelGGL((attn_fwd_kernel<DT, D>), dim3(tiles * a.n_heads * pc.most), dim3(256), 0, s, a, pc, tiles);
    if (pc.most > 1) hipLaunchKernelGGL((attn_fwd_join_kernel<DT, D>), dim3(tiles * 4, a.n_heads), dim3(256), 0, s, a, pc);
    return status_of(hipGetLastError());
}

template <int DT, int D>
int backward(const Attn &a, const Back &b, hipStream_t s) {
    const dim3 rows(b.blocks, a.n_heads + (DT == NF4_F16 ? a.n_kv : 0) + 1);
    const int groups = b.groups ? b.groups : b.tiles * (1 + a.group);
    hipLaunchKernelGGL((attn_rows_kernel<DT, D>), rows, dim3(256), 0, s, a, b);
    hipLaunchKernelGGL((attn_bwd_kernel<DT, D>), dim3(groups * a.n_kv), dim3(256), 0, s, a, b);
    if (b.groups > 1)
        hipLaunchKernelGGL((attn_bwd_join_kernel<DT, D>), dim3(8, b.groups * a.n_kv), dim3(256), 0, s, a, b);
    return status_of(hipGetLastError());
}

// out and stats as both passes have them
int take_saved(Attn &a, const nf4_attn *in, const void *out, const float *stats) {
    if (!out || !stats) return NF4_ERR_ARG;
    if (!aligned(out, 16) || !aligned(stats, 8)) return NF4_ERR_UNSUPPORTED;
    a.o = {static_cast<const uint16_t *>(out), static_cast<int64_t>(in->n_heads) * in->head_dim, in->head_dim};
    a.stats = reinterpret_cast<float2 *>(const_cast<float *>(stats));
    return NF4_OK;
}

// What a row of the longest sequence sees, as the host knows it.
int64_t span_of(const nf4_attn *in) {
    return in->max_len && in->max_len < in->tokens ? in->max_len : in->tokens;
}

// Steps of 64 of a tile of 128 rows (or keys): on average, and at most.
struct Steps {
    double mean;
    int64_t most;
};
Steps steps_of(const nf4_attn *in) {
    const int64_t span = span_of(in), w = in->window && in->window < span ? in->window : span;
    // (a tile's rows see w + 127 keys of a long sequence's middle, and half as many on average where
    // the window is all of it)
    const double seen = w < span ? static_cast<double>(w) : 0.5 * span;
    const int64_t all = tiles_of(in, kTile), most = (w + kOwn - 1) / kTile + 2;
    return {fmin(seen / kTile + 1.5, all), most < all ? most : all};
}

// A launch's time by measured constants (us, heads of 128, two workgroups on every CU; alone on a CU a
// workgroup takes half as long): a step of the forward pass, of a tile of keys and of a tile of rows,
// a workgroup's beginning and end, a launch that joins, and 64 KB written and read again.
constexpr double kFwdStep = 2.2, kKeyStep = 2.1, kRowStep = 3.1, kBegin = 9., kJoin = 5., kPart = 0.015;

// (heads of 64: half the products for the same exponentials, and three workgroups a CU)
double step_us(const nf4_attn *in, double us) { return in->head_dim == 128 ? us : 0.6 * us; }
int places_of(const nf4_attn *in) { return in->head_dim == 128 ? 512 : 768; }

// Time of a launch of `groups` workgroups that take `work` together and `longest` each at most.
double launch_us(const nf4_attn *in, double groups, double work, double longest) {
    const double begin = step_us(in, kBegin), places = places_of(in);
    // (the last to end find the card half empty, the less so the more there are)
    return groups <= places ? (begin + longest) * fmax(groups / places, 0.5)
                            : (work + groups * begin) / places + longest * places / groups / 2;
}

// The forward pass's launch, and the bytes of its workspace.
size_t plan(Pieces &p, const nf4_attn *in) {
    const int64_t items = static_cast<int64_t>(tiles_of(in, kOwn)) * in->n_heads;
    const Steps n = steps_of(in);
    const double step = step_us(in, kFwdStep);
    double best = INFINITY;
    for (double per = 4.; ; per *= 1.25) {
        const bool whole = per >= n.most;
        const double most = whole ? 1. : fmin(ceil(n.most / floor(per)), 64.), pieces = whole ? 1. : fmax(1., n.mean / per + 0.5);
        double t = launch_us(in, items * pieces, items * n.mean * step, fmin(per, n.most) * step);
        if (!whole) t += kJoin + items * pieces * kPart;
        if (t < best) {
            best = t;
            p.per = static_cast<int>(fmin(per, n.most));
            p.most = static_cast<int>(most);
        }
        if (whole) break;
    }
    return p.most > 1 ? items * p.most * kOwn * (in->head_dim * 4 + 8) : 0;
}

// The backward pass's launch, and its workspace, in bytes one behind the other from 0 on.
size_t plan(Back &b, const nf4_attn *in) {
    b.blocks = tiles_of(in, kTile);
    b.tiles = tiles_of(in, kOwn);
    const Steps n = steps_of(in);
    const int64_t rows = static_cast<int64_t>(b.tiles) * in->n_heads, keys = static_cast<int64_t>(b.tiles) * in->n_kv;
    const int64_t units = in->n_heads / in->n_kv * (kTile / kRows);  // steps of keys where rows have one
    const int places = places_of(in);
    const double key = step_us(in, kKeyStep), row = step_us(in, kRowStep);
    const double work = rows * n.mean * row + keys * n.mean * units * key;
    const double line = rows * n.mean * (kTile / kRows * kKeyCost + kRowCost) + (rows + keys) * kItemCost;
    const double groups = fmin(floor(line / kLeast), places);
    const double shares = (work + (rows + keys + groups) * step_us(in, kBegin)) / groups * fmax(groups / places, 0.5) +
                          kJoin + groups * kPart * in->head_dim / 64;
    const double most_keys = fmin(n.most * (kTile / kRows), tiles_of(in, kRows)) * (in->n_heads / in->n_kv);
    const double tiles = launch_us(in, rows + keys, work, fmax(n.most * row, most_keys * key));
    b.groups = shares < 1.1 * tiles || rows + keys > (1 << 23) ? static_cast<int>(fmax(groups / in->n_kv, 1.)) : 0;
    size_t at = 0;
    auto next = [&](size_t bytes) {
        char *p = reinterpret_cast<char *>(at);
        at += (bytes + 15) / 16 * 16;
        return p;
    };
    b.rows = reinterpret_cast<float *>(next(static_cast<size_t>(in->n_heads) * b.blocks * 1024));
    b.norms = reinterpret_cast<float *>(next(in->dtype == NF4_F16 ? static_cast<size_t>(2 * in->n_heads + in->n_kv) * b.blocks * 4 : 0));
    b.tab = reinterpret_cast<int4 *>(next(static_cast<size_t>(b.tiles) * 16));
    b.line = reinterpret_cast<int64_t *>(next((2 * static_cast<size_t>(b.tiles) + 1) * 8));
    b.inside = reinterpret_cast<int *>(next(static_cast<size_t>(b.groups) * in->n_kv * 4));
    const size_t slots = b.groups > 1 ? 2 * static_cast<size_t>(b.groups) * in->n_kv : 0;
    b.part = reinterpret_cast<float *>(next(slots * 2 * kOwn * in->head_dim * 4));
    return at;
}

}  // namespace

extern "C" size_t nf4_attn_fwd_workspace(const nf4_attn *in) {
    Attn a{};
    Pieces p{};
    return fill(a, in) != NF4_OK || in->tokens == 0 ? 0 : plan(p, in);
}

extern "C" int nf4_attn_fwd(const nf4_attn *in, void *out, float *stats, void *workspace,
                            size_t workspace_bytes, void *stream) {
    Attn a{};
    int st = fill(a, in);
    if (st != NF4_OK || in->tokens == 0) return st;
    if ((st = take_saved(a, in, out, stats)) != NF4_OK) return st;
    Pieces p{};
    const size_t need = plan(p, in);
    const int tiles = tiles_of(in, kOwn);
    if (need) {
        if (!workspace || workspace_bytes < need) return NF4_ERR_WORKSPACE;
        if (!aligned(workspace, 16)) return NF4_ERR_UNSUPPORTED;
        p.part = static_cast<float *>(workspace);
        p.ml = reinterpret_cast<float2 *>(p.part + static_cast<int64_t>(tiles) * in->n_heads * p.most * kOwn * in->head_dim);
    }
    auto s = static_cast<hipStream_t>(stream);
    if (in->dtype == NF4_BF16)
        return in->head_dim == 128 ? forward<NF4_BF16, 128>(a, p, tiles, s) : forward<NF4_BF16, 64>(a, p, tiles, s);
    return in->head_dim == 128 ? forward<NF4_F16, 128>(a, p, tiles, s) : forward<NF4_F16, 64>(a, p, tiles, s);
}

extern "C" size_t nf4_attn_bwd_workspace(const nf4_attn *in) {
    Attn a{};
    Back b{};
    return fill(a, in) != NF4_OK || in->tokens == 0 ? 0 : plan(b, in);
}

extern "C" int nf4_attn_bwd(const nf4_attn *in, const void *out, const float *stats,
                            const nf4_grad *dout, const nf4_grad *dq, const nf4_grad *dk,
                            const nf4_grad *dv, void *workspace, size_t workspace_bytes,
                            void *stream) {
    Attn a{};
    int st = fill(a, in);
    if (st != NF4_OK || in->tokens == 0) return st;
    if ((st = take_saved(a, in, out, stats)) != NF4_OK) return st;
    if (!dout) return NF4_ERR_ARG;
    if ((st = take(a.dout, dout->p, dout->tok, dout->head, in->tokens, in->n_heads)) != NF4_OK) return st;
    if ((st = take(a.dq, dq, in->tokens, in->n_heads, in->head_dim)) != NF4_OK) return st;
    if ((st = take(a.dk, dk, in->tokens, in->n_kv, in->head_dim)) != NF4_OK) return st;
    if ((st = take(a.dv, dv, in->tokens, in->n_kv, in->head_dim)) != NF4_OK) return st;
    Back b{};
    const size_t need = plan(b, in);
    if (!workspace || workspace_bytes < need) return NF4_ERR_WORKSPACE;
    if (!aligned(workspace, 16)) return NF4_ERR_UNSUPPORTED;
    auto moved = [&](auto *&p) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(static_cast<char *>(workspace) + reinterpret_cast<uintptr_t>(p));
    };
    moved(b.rows);
    moved(b.norms);
    moved(b.tab);
    moved(b.line);
    moved(b.inside);
    moved(b.part);
    auto s = static_cast<hipStream_t>(stream);
    if (in->dtype == NF4_BF16)
        return in->head_dim == 128 ? backward<NF4_BF16, 128>(a, b, s) : backward<NF4_BF16, 64>(a, b, s);
    return in->head_dim == 128 ? backward<NF4_F16, 128>(a, b, s) : backward<NF4_F16, 64>(a, b, s);
}
