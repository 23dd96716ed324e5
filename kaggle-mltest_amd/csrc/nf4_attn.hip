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

// The rows [s, e) of row t's sequence, or [t, t) of a row that belongs to none.
__device__ __forceinline__ int2 sequence_of(const Attn &a, int t) {
    if (!a.cu) return make_int2(0, a.tokens);
    int lo = 0, hi = a.batch + 1;  // the first offset past t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= t) lo = mid + 1;
        else hi = mid;
    }
    if (lo == 0 || lo > a.batch) return make_int2(t, t);
    const int s = a.cu[lo - 1], e = a.cu[lo];
    return make_int2(s < 0 ? 0 : s, e > a.tokens ? a.tokens : e);
}

// The keys [lo, hi) that row t sees, and the rows [t, hi) that see key t.
__device__ __forceinline__ int2 keys_of(const Attn &a, int t) {
    const int2 s = sequence_of(a, t);
    if (s.y <= t) return make_int2(t, t);
    return make_int2(a.window && t - a.window + 1 > s.x ? t - a.window + 1 : s.x, t + 1);
}
__device__ __forceinline__ int2 rows_of(const Attn &a, int t) {
    const int2 s = sequence_of(a, t);
    if (s.y <= t) return make_int2(t, t);
    return make_int2(t, a.window && t + a.window < s.y ? t + a.window : s.y);
}

// A score's exponent: fma(score, c, -m), exact but for its own rounding; where m is far from 0 the
// rounding of m itself would show in that (16 and more from 2^28 on), so there the product is rounded
// as m was.  Never above 0, where m is the largest: sums in another order could be.
constexpr float kFar = 1 << 20;
__device__ __forceinline__ float exponent(float s, float c, float m) {
    const float x = fabsf(m) > kFar ? s * c - m : fmaf(s, c, -m);
    return x > 0.f ? 0.f : x;  // (a NaN stays)
}

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

// acc += f * this lane's channels of a row
template <int DT, int D>
__device__ __forceinline__ void add_row(float (&acc)[D / 64], float f, const uint16_t *row) {
    const int l = threadIdx.x & 63;
    if constexpr (D == 128) {
        const uint32_t w = *reinterpret_cast<const uint32_t *>(row + 2 * l);
        acc[0] = fmaf(f, f32_of<DT>(w & 0xffffu), acc[0]);
        acc[1] = fmaf(f, f32_of<DT>(w >> 16), acc[1]);
    } else {
        acc[0] = fmaf(f, f32_of<DT>(row[l]), acc[0]);
    }
}

template <int DT, int D>
__device__ __forceinline__ void store_row(uint16_t *row, const float (&v)[D / 64]) {
    const int l = threadIdx.x & 63;
    if constexpr (D == 128)
        *reinterpret_cast<uint32_t *>(row + 2 * l) = round16<DT>(v[0]) | static_cast<uint32_t>(round16<DT>(v[1])) << 16;
    else row[l] = round16<DT>(v[0]);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// (m, l) of row r over keys [k0, k1), and acc = sum 2^(t - m) v
template <int DT, int D>
__device__ __forceinline__ void row_forward(const Attn &a, int head, int r, int k0, int k1, float &m,
                                            float &l, float (&acc)[D / 64]) {
    const int lane = threadIdx.x & 63, kvh = head / a.group;
    const uint16_t *q = a.q.at(r, head);
    m = -INFINITY;
    for (int k = k0; k < k1; k += 64)
        if (k + lane < k1) m = fmaxf(m, dot_of<DT, D>(q, a.k.at(k + lane, kvh)) * a.c);
    m = wave_max(m);
    l = 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] = 0.f;
    for (int k = k0; k < k1; k += 64) {
        float p = 0.f;
        if (k + lane < k1)
            p = __builtin_amdgcn_exp2f(exponent(dot_of<DT, D>(q, a.k.at(k + lane, kvh)), a.c, m));
        l += p;
        const int n = k1 - k < 64 ? k1 - k : 64;
        for (int i = 0; i < n; ++i) add_row<DT, D>(acc, lane_value(p, i), a.v.at(k + i, kvh));
    }
    l = wave_sum(l);
}

// acc = sum over keys [k0, k1) of dS k
template <int DT, int D>
__device__ __forceinline__ void row_backward(const Attn &a, int head, int r, int k0, int k1,
                                             float (&acc)[D / 64]) {
    const int lane = threadIdx.x & 63, kvh = head / a.group;
    const uint16_t *q = a.q.at(r, head), *go = a.dout.at(r, head);
    const float2 ml = a.stats[static_cast<int64_t>(r) * a.n_heads + head];
    const float delta = dot_of<DT, D>(go, a.o.at(r, head)), inv = 1.f / ml.y;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] = 0.f;
    for (int k = k0; k < k1; k += 64) {
        float ds = 0.f;
        if (k + lane < k1) {
            const float p = __builtin_amdgcn_exp2f(exponent(dot_of<DT, D>(q, a.k.at(k + lane, kvh)), a.c, ml.x)) * inv;
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
    const int lane = threadIdx.x & 63, kvh = head / a.group;
    const uint16_t *kj = a.k.at(j, kvh), *vj = a.v.at(j, kvh);
    for (int r = r0; r < r1; r += 64) {
        float p = 0.f, ds = 0.f;
        if (r + lane < r1) {
            const float2 ml = a.stats[static_cast<int64_t>(r + lane) * a.n_heads + head];
            const uint16_t *go = a.dout.at(r + lane, head);
            p = __builtin_amdgcn_exp2f(exponent(dot_of<DT, D>(kj, a.q.at(r + lane, head)), a.c, ml.x)) / ml.y;
            ds = p * (dot_of<DT, D>(vj, go) - dot_of<DT, D>(go, a.o.at(r + lane, head)));
        }
        const int n = r1 - r < 64 ? r1 - r : 64;
        for (int i = 0; i < n; ++i) {
            add_row<DT, D>(dv, lane_value(p, i), a.dout.at(r + i, head));
            add_row<DT, D>(dk, lane_value(ds, i), a.q.at(r + i, head));
        }
    }
}

template <int DT, int D>
__global__ __launch_bounds__(256) void attn_rows_kernel(const Attn a, int grad) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (i >= static_cast<int64_t>(a.tokens) * a.n_heads) return;
    const int r = __builtin_amdgcn_readfirstlane(static_cast<int>(i / a.n_heads));
    const int head = __builtin_amdgcn_readfirstlane(static_cast<int>(i % a.n_heads));
    const int2 seen = keys_of(a, r);
    float acc[D / 64], m = 0.f, l = 0.f;
    if (grad) {
        row_backward<DT, D>(a, head, r, seen.x, seen.y, acc);
#pragma unroll
        for (int x = 0; x < D / 64; ++x) acc[x] *= a.scale;
        store_row<DT, D>(a.dq.to(r, head), acc);
        return;
    }
    row_forward<DT, D>(a, head, r, seen.x, seen.y, m, l, acc);
    const bool none = seen.x == seen.y;
#pragma unroll
    for (int x = 0; x < D / 64; ++x) acc[x] = none ? 0.f : acc[x] / l;
    store_row<DT, D>(a.o.to(r, head), acc);
    if ((threadIdx.x & 63) == 0) a.stats[i] = none ? make_float2(0.f, 0.f) : make_float2(m, l);
}

template <int DT, int D>
__global__ __launch_bounds__(256) void attn_keys_kernel(const Attn a) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (i >= static_cast<int64_t>(a.tokens) * a.n_kv) return;
    const int j = __builtin_amdgcn_readfirstlane(static_cast<int>(i / a.n_kv));
    const int kvh = __builtin_amdgcn_readfirstlane(static_cast<int>(i % a.n_kv));
    const int2 seen = rows_of(a, j);
    float dk[D / 64] = {}, dv[D / 64] = {};
    for (int h = 0; h < a.group; ++h)
        key_backward<DT, D>(a, kvh * a.group + h, j, seen.x, seen.y, dk, dv);
#pragma unroll
    for (int x = 0; x < D / 64; ++x) dk[x] *= a.scale;
    store_row<DT, D>(a.dk.to(j, kvh), dk);
    store_row<DT, D>(a.dv.to(j, kvh), dv);
}

// ------------------------------------------------------------------------- host

struct Shape {
    int head_dim, dtype;
};

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

dim3 waves(int64_t n) { return dim3(static_cast<unsigned>((n + 3) / 4)); }

template <int DT, int D>
int launch(const Attn &a, bool grad, hipStream_t s) {
    const int64_t rows = static_cast<int64_t>(a.tokens) * a.n_heads, keys = static_cast<int64_t>(a.tokens) * a.n_kv;
    hipLaunchKernelGGL((attn_rows_kernel<DT, D>), waves(rows), dim3(256), 0, s, a, grad ? 1 : 0);
    if (grad) hipLaunchKernelGGL((attn_keys_kernel<DT, D>), waves(keys), dim3(256), 0, s, a);
    return status_of(hipGetLastError());
}

int launch_of(const Attn &a, const nf4_attn *in, bool grad, hipStream_t s) {
    if (in->dtype == NF4_BF16)
        return in->head_dim == 128 ? launch<NF4_BF16, 128>(a, grad, s) : launch<NF4_BF16, 64>(a, grad, s);
    return in->head_dim == 128 ? launch<NF4_F16, 128>(a, grad, s) : launch<NF4_F16, 64>(a, grad, s);
}

// out and stats as both passes have them
int take_saved(Attn &a, const nf4_attn *in, const void *out, const float *stats) {
    if (!out || !stats) return NF4_ERR_ARG;
    if (!aligned(out, 16) || !aligned(stats, 8)) return NF4_ERR_UNSUPPORTED;
    a.o = {static_cast<const uint16_t *>(out), static_cast<int64_t>(in->n_heads) * in->head_dim, in->head_dim};
    a.stats = reinterpret_cast<float2 *>(const_cast<float *>(stats));
    return NF4_OK;
}

}  // namespace

extern "C" size_t nf4_attn_fwd_workspace(const nf4_attn *in) { return 0; }

extern "C" int nf4_attn_fwd(const nf4_attn *in, void *out, float *stats, void *workspace,
                            size_t workspace_bytes, void *stream) {
    Attn a{};
    int st = fill(a, in);
    if (st != NF4_OK || in->tokens == 0) return st;
    if ((st = take_saved(a, in, out, stats)) != NF4_OK) return st;
    return launch_of(a, in, false, static_cast<hipStream_t>(stream));
}

extern "C" size_t nf4_attn_bwd_workspace(const nf4_attn *in) { return 0; }

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
    return launch_of(a, in, true, static_cast<hipStream_t>(stream));
}
