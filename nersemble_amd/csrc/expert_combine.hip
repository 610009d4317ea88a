// expert_combine.hip -- routed experts: the weighted join of a row's expert outputs, and its gradients.
//
// out_t = sum_j w_tj y_pos(t,j);  dy_pos(t,j) = w_tj dout_t;  dw_tj = <dout_t, y_pos(t,j)>.  Sums in 32 bits; each result is rounded
// to 16 bits once (dy: one product, rounded).
// Bound by memory: y is read once, by rows of the plan's order, out or dy written once.  us and bytes / time of calls repeated on the
// same arrays, which the last-level cache partly holds (with other data in between 8192 x 8 takes 41 and 57):
//   262144 rows x 2 choices, 64 columns fp16     forward 19.6 (105 MB, 5.4 TB/s)   backward 35.7 (174 MB, 4.9 TB/s)
//   8192 x 8, 1024 columns bf16                  forward 30.4 (151 MB, 5.0 TB/s)   backward 63 (286 MB, 4.5 TB/s; a copy 4.96)
//   524289 x 2, 16 columns fp16                                                    backward 22.8 (96 MB, 4.2 TB/s)
// Stores past the caches (nontemporal) took 17, 32, 28.6 and 60 us (the first two lines), but the next reader of the result pays what they gain.
#include "expert_common.h"

namespace nsx {

struct CombineArgs {
    const void* y; int64_t y_stride;
    const float* w;                  // NULL: every weight is 1
    const int32_t* positions; const int32_t* offsets;
    int64_t T; int k, R, chunks;     // chunks: 8-wide pieces of a row
    const int64_t* n_dev;
};

__device__ __forceinline__ int64_t valid_rows(int64_t T, const int64_t* n_dev) {
    if (!n_dev) return T;
    const int64_t n = *n_dev;
    return n < T ? (n < 0 ? 0 : n) : T;
}

// A thread makes 8 columns of a row (16 bytes per load and store, neighbours side by side); the KU choices of a round are read side
// by side, so that their latencies overlap, and added in their order: 8 choices one after the other take 34 us where this takes 30.
// Y: what y lies in (the type of the result, or 32 bits).
template <typename T, int KU, typename Y>
__global__ __launch_bounds__(256) void combine_fwd_kernel(CombineArgs a, T* __restrict__ out) {
    typedef typename Elem<T>::x8 x8;
    typedef typename Elem<Y>::x8 y8;
    const int64_t total = valid_rows(a.T, a.n_dev) * a.chunks;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / a.chunks;
        const int c = (int)(i - t * a.chunks);
        float s[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) s[q] = 0.f;
        for (int j = 0; j < a.k; j += KU) {
            int p[KU];
            float w[KU];
            y8 v[KU];
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                const bool in = KU <= 2 || j + u < a.k;
                p[u] = in ? a.positions[t * a.k + j + u] : -1;
                w[u] = in && a.w ? a.w[t * a.k + j + u] : 1.f;
            }
#pragma unroll
            for (int u = 0; u < KU; ++u)
                if ((unsigned)p[u] < (unsigned)a.R) v[u] = *reinterpret_cast<const y8*>(reinterpret_cast<const Y*>(a.y) + (int64_t)p[u] * a.y_stride + c * 8);
#pragma unroll
            for (int u = 0; u < KU; ++u)
                if ((unsigned)p[u] < (unsigned)a.R)
#pragma unroll
                    for (int q = 0; q < 8; ++q) s[q] += w[u] * (float)v[u][q];
        }
        x8 o;
#pragma unroll
        for (int q = 0; q < 8; ++q) o[q] = (T)s[q];
        *reinterpret_cast<x8*>(out + i * 8) = o;
    }
}

// 2^lg lanes per row of `out`: y is read once, dy written once, dout once or (from the caches) once per choice; the
// products' sum goes through the row's lanes in a fixed order, no atomics.
// CP: pieces of a row that a lane keeps in registers (0: any number, dout read again for every choice); KU: choices side by side.
template <typename T, int CP, int KU>
__global__ __launch_bounds__(256) void combine_bwd_kernel(CombineArgs a, const T* __restrict__ dout, T* __restrict__ dy,
                                                          float* __restrict__ dw, int lg) {
    typedef typename Elem<T>::x8 x8;
    const int lanes = 1 << lg, sub = threadIdx.x & (lanes - 1);
    const int64_t T_ = valid_rows(a.T, a.n_dev);
    const int64_t step = ((int64_t)gridDim.x * 256) >> lg;
    for (int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> lg; t < T_; t += step) {
        x8 g[CP > 0 ? CP : 1];
#pragma unroll
        for (int i = 0; i < CP; ++i) {
            const int c = sub + i * lanes;
            if (c < a.chunks) g[i] = *reinterpret_cast<const x8*>(dout + (t * a.chunks + c) * 8);
        }
        for (int j = 0; j < a.k; j += KU) {
            int p[KU];
            float w[KU], dot[KU];
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                const bool in = KU == 1 || j + u < a.k;
                p[u] = in ? a.positions[t * a.k + j + u] : -1;
                w[u] = in ? a.w[t * a.k + j + u] : 0.f;
                dot[u] = 0.f;
            }
            auto piece = [&](int u, int c, x8 g, x8 v) {
                x8 o;
#pragma unroll
                for (int q = 0; q < 8; ++q) { dot[u] += (float)g[q] * (float)v[q]; o[q] = (T)(w[u] * (float)g[q]); }
                *reinterpret_cast<x8*>(dy + ((int64_t)p[u] * a.chunks + c) * 8) = o;
            };
            auto read = [&](int u, int c) { return *reinterpret_cast<const x8*>(reinterpret_cast<const T*>(a.y) + (int64_t)p[u] * a.y_stride + c * 8); };
            if (CP > 0) {
                x8 v[KU][CP > 0 ? CP : 1];
#pragma unroll
                for (int u = 0; u < KU; ++u)
                    if ((unsigned)p[u] < (unsigned)a.R)
#pragma unroll
                        for (int i = 0; i < CP; ++i) if (sub + i * lanes < a.chunks) v[u][i] = read(u, sub + i * lanes);
#pragma unroll
                for (int u = 0; u < KU; ++u)
                    if ((unsigned)p[u] < (unsigned)a.R)
#pragma unroll
                        for (int i = 0; i < CP; ++i) if (sub + i * lanes < a.chunks) piece(u, sub + i * lanes, g[i], v[u][i]);
            } else if ((unsigned)p[0] < (unsigned)a.R) {
                for (int c = sub; c < a.chunks; c += lanes)
                    piece(0, c, *reinterpret_cast<const x8*>(dout + (t * a.chunks + c) * 8), read(0, c));
            }
#pragma unroll
            for (int u = 0; u < KU; ++u) {
                for (int o = 1; o < lanes; o <<= 1) dot[u] += __shfl_xor(dot[u], o);
                if (sub == 0 && j + u < a.k) dw[t * a.k + j + u] = (unsigned)p[u] < (unsigned)a.R ? dot[u] : 0.f;
            }
        }
    }
    // rows of dy behind the last segment
    const int64_t first = (int64_t)min(max(*a.offsets, 0), a.R) * a.chunks, last = (int64_t)a.R * a.chunks;
    x8 z;
#pragma unroll
    for (int q = 0; q < 8; ++q) z[q] = (T)0.f;
    for (int64_t i = first + (int64_t)blockIdx.x * 256 + threadIdx.x; i < last; i += (int64_t)gridDim.x * 256)
        *reinterpret_cast<x8*>(dy + i * 8) = z;
}

template <typename T>
static void combine_bwd_launch(const CombineArgs& a, const T* dout, T* dy, float* dw, int lg, unsigned grid, hipStream_t st) {
    // us, dout read for every choice | kept, two choices at a time: rows of 16 columns, 524289 x 2  28.8 | 22.7, of 64, 262144 x 2
    // 35.2 | 36.0, of 512, 4096 x 4  8.6 | 9.1, of 520, 20000 x 3  37.1 | 38.1, of 1024, 8192 x 8  65.5 | 63.1, of 2048, 16384 x 2  68.2 | 71.3
    if (lg <= 2) combine_bwd_kernel<T, 1, 2><<<grid, 256, 0, st>>>(a, dout, dy, dw, lg);
    else if (a.chunks > 96 && a.chunks <= 128) combine_bwd_kernel<T, 2, 2><<<grid, 256, 0, st>>>(a, dout, dy, dw, lg);
    else combine_bwd_kernel<T, 0, 1><<<grid, 256, 0, st>>>(a, dout, dy, dw, lg);
}
template <typename Y, typename T>
static void combine_fwd_launch(const CombineArgs& a, T* out, hipStream_t st) {
    const int64_t blocks = (a.T * a.chunks + 255) / 256, most = (int64_t)num_cus() * 32;
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    if (a.k == 1) combine_fwd_kernel<T, 1, Y><<<grid, 256, 0, st>>>(a, out);
    else if (a.k == 2) combine_fwd_kernel<T, 2, Y><<<grid, 256, 0, st>>>(a, out);
    else combine_fwd_kernel<T, 4, Y><<<grid, 256, 0, st>>>(a, out);
}

int expert_join_f32(const float* y, int64_t R, int n, const int32_t* positions, int64_t T, int top_k, void* out, int dtype, hipStream_t st) {
    if (T == 0) return NSX_OK;
    const CombineArgs a{y, n, nullptr, positions, nullptr, T, top_k, (int)R, n / 8, nullptr};
    if (dtype == NSX_DTYPE_F16) combine_fwd_launch<float>(a, (half_t*)out, st);
    else combine_fwd_launch<float>(a, (bf16_t*)out, st);
    NSX_LAUNCH_CHECK("expert_join_f32");
    return NSX_OK;
}

}  // namespace nsx

extern "C" {

static int combine_check(const char* what, int dtype, int64_t T, int top_k, int64_t R, int n, int64_t stride, const void* y) {
    using namespace nsx;
    NSX_REQUIRE(dtype == NSX_DTYPE_F16 || dtype == NSX_DTYPE_BF16, "%s: dtype %d is not a 16-bit float", what, dtype);
    NSX_REQUIRE(top_k >= 1 && top_k <= NSX_MAX_TOP_K, "%s: top_k %d not in [1,%d]", what, top_k, NSX_MAX_TOP_K);
    NSX_REQUIRE(T >= 0 && T <= NSX_MAX_EXPERT_ENTRIES / top_k, "%s: %lld rows of %d choices are too many", what, (long long)T, top_k);
    NSX_REQUIRE(R >= 0 && R <= NSX_MAX_EXPERT_ENTRIES, "%s: %lld ordered rows", what, (long long)R);
    NSX_REQUIRE(n >= 8 && n % 8 == 0 && n <= NSX_MAX_EXPERT_WIDTH, "%s: width %d is not a multiple of 8 in [8,%d]", what, n, NSX_MAX_EXPERT_WIDTH);
    NSX_REQUIRE(stride >= n && stride % 8 == 0 && aligned16(y), "%s: rows of y are not 16-byte aligned (stride %lld)", what, (long long)stride);
    return NSX_OK;
}

int nsx_expert_combine_fwd(const void* y, int dtype, int64_t y_stride, int64_t R, int n, const float* weights,
                           const int32_t* positions, int64_t T, int top_k, void* out, const int64_t* n_device, void* stream) {
    using namespace nsx;
    const int rc = combine_check("nsx_expert_combine_fwd", dtype, T, top_k, R, n, y_stride, y);
    if (rc != NSX_OK) return rc;
    if (T == 0) return NSX_OK;
    NSX_REQUIRE(positions && out && (y || R == 0) && aligned16(out), "nsx_expert_combine_fwd: NULL or unaligned pointer");
    CombineArgs a{y, y_stride, weights, positions, nullptr, T, top_k, (int)R, n / 8, n_device};
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NSX_DTYPE_F16) combine_fwd_launch<half_t>(a, (half_t*)out, st);
    else combine_fwd_launch<bf16_t>(a, (bf16_t*)out, st);
    NSX_LAUNCH_CHECK("nsx_expert_combine_fwd");
    return NSX_OK;
}

int nsx_expert_combine_bwd(const void* y, int dtype, int64_t y_stride, int64_t R, int n, const float* weights,
                           const int32_t* positions, const int32_t* n_routed, int64_t T, int top_k, const void* dout, void* dy,
                           float* dweights, const int64_t* n_device, void* stream) {
    using namespace nsx;
    const int rc = combine_check("nsx_expert_combine_bwd", dtype, T, top_k, R, n, y_stride, y);
    if (rc != NSX_OK) return rc;
    if (T == 0 && R == 0) return NSX_OK;
    NSX_REQUIRE(n_routed && (T == 0 || (weights && positions && dout && dweights && aligned16(dout))) && (R == 0 || (y && dy && aligned16(dy))),
                "nsx_expert_combine_bwd: NULL or unaligned pointer");
    CombineArgs a{y, y_stride, weights, positions, n_routed, T, top_k, (int)R, n / 8, n_device};
    int lg = 0;
    while ((1 << lg) < n / 8 && lg < 6) ++lg;
    const int64_t blocks = ((T << lg) + 255) / 256, most = (int64_t)num_cus() * 32;
    const unsigned grid = (unsigned)(blocks < 1 ? 1 : blocks < most ? blocks : most);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NSX_DTYPE_F16)
        combine_bwd_launch(a, (const half_t*)dout, (half_t*)dy, dweights, lg, grid, st);
    else
        combine_bwd_launch(a, (const bf16_t*)dout, (bf16_t*)dy, dweights, lg, grid, st);
    NSX_LAUNCH_CHECK("nsx_expert_combine_bwd");
    return NSX_OK;
}

}  // extern "C"
