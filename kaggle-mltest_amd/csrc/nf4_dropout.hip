// Dropout from a counter-based generator, for gfx950: LoRA's dropped inputs without a stored mask.
//
// An element's number is a function of its place, the site's number and the step's, so the backward
// pass forms the mask again instead of reading one.  Philox4x32-10 (Salmon, Moraes, Dror, Shaw,
// "Parallel random numbers: as easy as 1, 2, 3", 2011): ten rounds on a counter of four 32-bit
// words, each round two 32 x 32 -> 64-bit products whose high halves are mixed with the other words
// and the key.  The counter is (group lo, group hi, step, site) and the key the 64-bit seed; group
// row * ceil(cols / 8) + col / 8 are eight columns of a row, whose numbers are the eight 16-bit
// halves of the result.  An element is kept where its number is at least T = round(65536 p), and
// scaled by 65536 / (65536 - T), the share that is kept: the mean is exact for every T.
//
// A thread takes one group for every site of the call, so that x (or the sum) is read once for all
// of a layer's adapters.  Bound by memory: 8192 x 3584, two sites, bf16: 29.7 us, 5.9 TB/s, its gradient 37.6,
// 6.2; seven sites 89 and 104 us, 5.2.  Widths that are no multiple of 8, or rows off 16 bytes, go a value at a
// time: 8192 x 3583 takes 100 and 118 us, three times as long.

#include "nf4_common.h"

namespace {

constexpr int kDropThreads = 256, kDropSites = 8;

struct Drop {
    const uint16_t *in[kDropSites];  // the input (one), or the sites' gradients
    uint16_t *out[kDropSites];       // the sites' outputs, or the sum (one)
    int64_t ld_in[kDropSites], ld_out[kDropSites];
    uint32_t site[kDropSites];
    const uint16_t *base;            // added to the gradients' sum, or null
    int64_t ld_base;
    const int64_t *seed;             // device: seed, step
    uint32_t groups, per, cols;      // of eight columns: all, of a row
    uint32_t cut;                    // T
    float scale;
};

// The eight 16-bit numbers of a group.
__device__ __forceinline__ u32x4_t philox(uint32_t g, uint32_t step, uint32_t site, uint32_t k0,
                                          uint32_t k1) {
    uint32_t a = g, b = 0, c = step, d = site;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t x = static_cast<uint64_t>(a) * 0xD2511F53u;
        const uint64_t y = static_cast<uint64_t>(c) * 0xCD9E8D57u;
        a = static_cast<uint32_t>(y >> 32) ^ b ^ k0;
        b = static_cast<uint32_t>(y);
        c = static_cast<uint32_t>(x >> 32) ^ d ^ k1;
        d = static_cast<uint32_t>(x);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return (u32x4_t){a, b, c, d};
}

// Columns [c, c + 8) of a row of `cols`: 16 bytes where VEC (every row 16-byte aligned), and one
// value at a time where it is not, or at a row's end.
template <bool VEC>
__device__ __forceinline__ u32x4_t load_group(const uint16_t *p, int c, int cols) {
    if (VEC && c + 8 <= cols) return *reinterpret_cast<const u32x4_t *>(p + c);
    u32x4_t r = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < cols) r[i >> 1] |= static_cast<uint32_t>(p[c + i]) << (16 * (i & 1));
    return r;
}

template <bool VEC>
__device__ __forceinline__ void store_group(uint16_t *p, int c, int cols, const u32x4_t &v) {
    if (VEC && c + 8 <= cols) {
        *reinterpret_cast<u32x4_t *>(p + c) = v;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (c + i < cols) p[c + i] = static_cast<uint16_t>(v[i >> 1] >> (16 * (i & 1)));
}

template <int DT, int N, bool VEC>
__global__ __launch_bounds__(kDropThreads) void dropout_kernel(const Drop a) {
    const uint32_t g = blockIdx.x * kDropThreads + threadIdx.x;
    if (g >= a.groups) return;
    const uint32_t row = g / a.per, cols = a.cols, c = (g - row * a.per) * 8;
    const uint64_t seed = a.seed[0];
    const uint32_t step = static_cast<uint32_t>(a.seed[1]);
    const uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
    float x[8];
    unpack8<DT>(load_group<VEC>(a.in[0] + row * a.ld_in[0], c, cols), x);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= a.scale;
#pragma unroll
    for (int s = 0; s < N; ++s) {
        const u32x4_t n = philox(g, step, a.site[s], k0, k1);
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (n[i >> 1] >> (16 * (i & 1)) & 0xffffu) >= a.cut ? x[i] : 0.f;
        store_group<VEC>(a.out[s] + row * a.ld_out[s], c, cols, pack8<DT>(y));
    }
}

// The sum in fp32, base first and the sites in their order; one rounding.
template <int DT, int N, bool VEC>
__global__ __launch_bounds__(kDropThreads) void dropout_bwd_kernel(const Drop a) {
    const uint32_t g = blockIdx.x * kDropThreads + threadIdx.x;
    if (g >= a.groups) return;
    const uint32_t row = g / a.per, cols = a.cols, c = (g - row * a.per) * 8;
    const uint64_t seed = a.seed[0];
    const uint32_t step = static_cast<uint32_t>(a.seed[1]);
    const uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
    u32x4_t in[N];
#pragma unroll
    for (int s = 0; s < N; ++s) in[s] = load_group<VEC>(a.in[s] + row * a.ld_in[s], c, cols);
    float sum[8];
    u32x4_t b = {0, 0, 0, 0};
    if (a.base) b = load_group<VEC>(a.base + row * a.ld_base, c, cols);
    unpack8<DT>(b, sum);
#pragma unroll
    for (int s = 0; s < N; ++s) {
        const u32x4_t n = philox(g, step, a.site[s], k0, k1);
        float x[8];
        unpack8<DT>(in[s], x);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            sum[i] += (n[i >> 1] >> (16 * (i & 1)) & 0xffffu) >= a.cut ? x[i] * a.scale : 0.f;
    }
    store_group<VEC>(a.out[0] + row * a.ld_out[0], c, cols, pack8<DT>(sum));
}

template <int DT, int N, bool VEC>
void launch(const Drop &a, bool grad, hipStream_t s) {
    const dim3 grid((a.groups + kDropThreads - 1) / kDropThreads);
    if (grad) hipLaunchKernelGGL((dropout_bwd_kernel<DT, N, VEC>), grid, dim3(kDropThreads), 0, s, a);
    else hipLaunchKernelGGL((dropout_kernel<DT, N, VEC>), grid, dim3(kDropThreads), 0, s, a);
}

template <int DT, bool VEC>
void launch_n(const Drop &a, int n, bool grad, hipStream_t s) {
    switch (n) {
    case 1: return launch<DT, 1, VEC>(a, grad, s);
    case 2: return launch<DT, 2, VEC>(a, grad, s);
    case 3: return launch<DT, 3, VEC>(a, grad, s);
    case 4: return launch<DT, 4, VEC>(a, grad, s);
    case 5: return launch<DT, 5, VEC>(a, grad, s);
    case 6: return launch<DT, 6, VEC>(a, grad, s);
    case 7: return launch<DT, 7, VEC>(a, grad, s);
    default: return launch<DT, 8, VEC>(a, grad, s);
    }
}

// What both calls check; `in` and `out` are n or one tensors.
int fill(Drop &a, const void *const *in, const int64_t *ld_in, int n_in, void *const *out,
         const int64_t *ld_out, int n_out, int64_t rows, int64_t cols, double p, const int64_t *seed,
         const uint32_t *sites, int n, int dtype, bool &vec) {
    if (dtype != NF4_F16 && dtype != NF4_BF16) return NF4_ERR_ARG;
    if (rows < 0 || cols < 0 || n < 1 || !in || !out || !ld_in || !ld_out || !sites) return NF4_ERR_ARG;
    if (!(p >= 0. && p <= 1.)) return NF4_ERR_ARG;  // NaN too
    if (n > kDropSites) return NF4_ERR_UNSUPPORTED;
    if (rows == 0 || cols == 0) return NF4_OK;
    if (!seed || !aligned(seed, 8)) return NF4_ERR_ARG;
    const int64_t per = (cols + 7) / 8;
    if (cols > 0x7fffffff - 8 || rows > 0x7fffffff || rows * per > 0x7fffffff - kDropThreads)
        return NF4_ERR_UNSUPPORTED;
    auto ok = [&](const void *t, int64_t ld) {
        if (!t || (rows > 1 && ld < cols)) return false;
        vec = vec && aligned(t, 16) && ld % 8 == 0;
        return true;
    };
    vec = true;
    for (int i = 0; i < n_in; ++i) {
        if (!ok(in[i], ld_in[i])) return NF4_ERR_ARG;
        a.in[i] = static_cast<const uint16_t *>(in[i]);
        a.ld_in[i] = ld_in[i];
    }
    for (int i = 0; i < n_out; ++i) {
        if (!ok(out[i], ld_out[i])) return NF4_ERR_ARG;
        a.out[i] = static_cast<uint16_t *>(out[i]);
        a.ld_out[i] = ld_out[i];
    }
    if (a.base && !ok(a.base, a.ld_base)) return NF4_ERR_ARG;
    for (int i = 0; i < n_in; ++i)
        if (!aligned(in[i], 2)) return NF4_ERR_ARG;
    for (int i = 0; i < n_out; ++i)
        if (!aligned(out[i], 2)) return NF4_ERR_ARG;
    if (!aligned(a.base, 2)) return NF4_ERR_ARG;
    for (int i = 0; i < n; ++i) a.site[i] = sites[i];
    a.seed = seed;
    a.per = static_cast<uint32_t>(per);
    a.cols = static_cast<uint32_t>(cols);
    a.groups = static_cast<uint32_t>(rows * per);
    a.cut = static_cast<uint32_t>(p * 65536. + 0.5);
    // (nothing is kept: any finite scale)
    a.scale = a.cut < 65536 ? 65536.f / static_cast<float>(65536 - a.cut) : 0.f;
    return NF4_OK;
}

int run(const Drop &a, int n, bool grad, bool vec, int dtype, void *stream) {
    if (a.groups == 0) return NF4_OK;
    auto s = static_cast<hipStream_t>(stream);
    if (dtype == NF4_BF16) vec ? launch_n<NF4_BF16, true>(a, n, grad, s) : launch_n<NF4_BF16, false>(a, n, grad, s);
    else vec ? launch_n<NF4_F16, true>(a, n, grad, s) : launch_n<NF4_F16, false>(a, n, grad, s);
    return status_of(hipGetLastError());
}

}  // namespace

extern "C" int nf4_dropout(const void *x, int64_t ld_x, void *const *outs, const int64_t *ld_outs,
                           int64_t rows, int64_t cols, double p, const int64_t *seed,
                           const uint32_t *sites, int n, int dtype, void *stream) {
    Drop a{};
    bool vec = false;
    const int st = fill(a, &x, &ld_x, 1, outs, ld_outs, n, rows, cols, p, seed, sites, n, dtype, vec);
    return st != NF4_OK ? st : run(a, n, false, vec, dtype, stream);
}

extern "C" int nf4_dropout_bwd(const void *const *grads, const int64_t *ld_grads, const void *base,
                               int64_t ld_base, void *dx, int64_t ld_dx, int64_t rows, int64_t cols,
                               double p, const int64_t *seed, const uint32_t *sites, int n, int dtype,
                               void *stream) {
    Drop a{};
    bool vec = false;
    a.base = static_cast<const uint16_t *>(base);
    a.ld_base = ld_base;
    const int st = fill(a, grads, ld_grads, n, &dx, &ld_dx, 1, rows, cols, p, seed, sites, n, dtype, vec);
    return st != NF4_OK ? st : run(a, n, true, vec, dtype, stream);
}
