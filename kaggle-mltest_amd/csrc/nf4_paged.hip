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

struct Query {
    const uint16_t *q;
    int64_t ld_tok, ld_head;
    uint16_t *out;
    float *lse;
    int n_heads, window, sinks, shared;
    float scale;
};

// One wave per (token, query head): 64 keys at a time, a lane per key for the scores, running
// maximum and sum, a lane per D / 64 channels for the products with v.
template <int DT, int D>
__global__ __launch_bounds__(64) void paged_attn_row_kernel(const Cache c, const Query a) {
    __shared__ float s_q[D];
    __shared__ float s_p[64];
    __shared__ int64_t s_at[64];
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const int b = seq_of_token(c, t), kvh = h / (a.n_heads / c.n_kv);
    const Seq s = seq_at(c, b);
    const int p = s.p0 + t - s.q0;
    for (int i = lane; i < D; i += 64) s_q[i] = f32_of<DT>(a.q[t * a.ld_tok + h * a.ld_head + i]);
    __syncthreads();
    const int end = p + 1 < c.cap ? p + 1 : c.cap;
    const int first = a.window && p - a.window + 1 > 0 ? p - a.window + 1 : 0;
    float m = -INFINITY, l = 0.f, o[D / 64] = {};
    int j0 = 0;
    while (j0 < end) {
        const int j = j0 + lane;
        int64_t at = -1;
        if (j < end && (j >= first || j < a.sinks)) at = slot_of(c, j < a.shared ? 0 : b, j);
        float sc = -INFINITY;
        if (at >= 0) {
            const uint16_t *kr = c.k + at + kvh * c.head_stride;
            sc = 0.f;
            for (int i = 0; i < D; i += 8) {
                float kk[8];
                unpack8<DT>(*reinterpret_cast<const u32x4_t *>(kr + i), kk);
#pragma unroll
                for (int e = 0; e < 8; ++e) sc += s_q[i + e] * kk[e];
            }
            sc *= a.scale;
        }
        float top = sc;
        for (int o2 = 32; o2; o2 >>= 1) top = fmaxf(top, __shfl_xor(top, o2));
        const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.f : mn;
        const float alpha = expf(m - base), pj = expf(sc - base);
        float sum = pj;
        for (int o2 = 32; o2; o2 >>= 1) sum += __shfl_xor(sum, o2);
        l = l * alpha + sum;
        m = mn;
        s_p[lane] = pj;
        s_at[lane] = at;
        __syncthreads();
        for (int i = 0; i < D / 64; ++i) {
            float acc = o[i] * alpha;
            for (int k = 0; k < 64; ++k)
                if (s_at[k] >= 0)
                    acc += s_p[k] * f32_of<DT>(c.v[s_at[k] + kvh * c.head_stride + i * 64 + lane]);
            o[i] = acc;
        }
        __syncthreads();
        j0 += 64;
        if (j0 >= a.sinks && j0 + 64 <= first) j0 = first & ~63;
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    for (int i = 0; i < D / 64; ++i)
        a.out[(static_cast<int64_t>(t) * a.n_heads + h) * D + i * 64 + lane] = round16<DT>(o[i] * inv);
    if (a.lse && lane == 0) a.lse[static_cast<int64_t>(t) * a.n_heads + h] = l > 0.f ? m + logf(l) : -INFINITY;
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
    c.cap = kv->width * kv->page_size;
    c.batch = kv->batch;
    c.n_kv = kv->n_kv;
    c.tokens = static_cast<int>(tokens);
    c.uniform = kv->batch ? static_cast<int>(tokens / kv->batch) : 0;
    return NF4_OK;
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
    return 0;
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
    auto cut = [](int64_t v) { return static_cast<int>(v < (1 << 30) ? v : 1 << 30); };
    Query a{};
    a.q = static_cast<const uint16_t *>(q);
    a.ld_tok = ld_tok;
    a.ld_head = ld_head;
    a.out = static_cast<uint16_t *>(out);
    a.lse = lse;
    a.n_heads = n_heads;
    a.window = cut(window);
    a.sinks = cut(sinks);
    a.shared = cut(shared);
    a.scale = scale;
    auto s = static_cast<hipStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(tokens), static_cast<unsigned>(n_heads));
#define NF4_ROW(DT, D) hipLaunchKernelGGL((paged_attn_row_kernel<DT, D>), grid, dim3(64), 0, s, c, a)
    if (dtype == NF4_BF16) {
        if (kv->head_dim == 64) NF4_ROW(NF4_BF16, 64);
        else NF4_ROW(NF4_BF16, 128);
    } else {
        if (kv->head_dim == 64) NF4_ROW(NF4_F16, 64);
        else NF4_ROW(NF4_F16, 128);
    }
#undef NF4_ROW
    return status_of(hipGetLastError());
}
