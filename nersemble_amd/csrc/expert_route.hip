// expert_route.hip -- routed experts: the choice of experts for every row, its gradient, and the plan that orders the
// (row, choice) entries by expert.
//
// Choice.  s_e = softmax(x)_e or 1 / (1 + exp(-x_e)); c_e = s_e + bias_e is what the choice goes by (the bias balances the
// experts' load and has no part in the weights).  With groups, a group counts for the sum of its `group_top` largest c, the
// `top_groups` best groups stay.  The top_k largest c that stay, in falling order, equal values by rising index, are the
// choice; w_j = scale * s_j / sum_i s_i (renormalised) or scale * s_j.
//   * Without a bias (and with groups that count for their largest c) the order of c IS the order of x: the logits are
//     compared as they are and no score is formed for experts that are not chosen.
//   * Otherwise c is formed in 64 bits: two experts whose 32-bit sums round to the same value, or change places, would make
//     the choice depend on the order of the summation behind the softmax.
//   * Renormalised weights are ratios: of the softmax only exp(x_j - max over the chosen) is left, of the sigmoid
//     exp(x_j - min(max, 0)) / (1 + exp(x_j)) -- neither underflows where all chosen scores are tiny.
// A row is held by L lanes of a wave, V consecutive experts in each (64 / L rows per wave): a row is read once, 16 bytes per
// lane, and the k rounds of "largest value, lowest index" are log2(L) exchanges each.
#include "expert_common.h"

namespace nsx {

struct RouteArgs {
    const void* x; int64_t stride; int64_t T; int E;
    const float* bias; const uint8_t* selector;
    int k, G, top_groups, group_top, sigmoid, renorm; float scale;
    float* w; int32_t* idx; const int64_t* n_dev;
    int lg_L, lg_Lg;                 // lanes per row and per group of it, as powers of two
};

constexpr int ROUTE_WAVES = 4;

template <typename T, int V, bool VEC>
__device__ __forceinline__ void load_logits(const T* __restrict__ p, int n, float (&x)[V]) {
    if (VEC) {
        struct alignas(sizeof(T) * V) Pack { T v[V]; };
        if (n > 0) {
            const Pack q = *reinterpret_cast<const Pack*>(p);
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = (float)q.v[i];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = -INFINITY;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = i < n ? (float)p[i] : -INFINITY;
    }
}

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }

template <typename K>
__device__ __forceinline__ K row_max(K v, int L) {
    for (int o = 1; o < L; o <<= 1) { const K u = __shfl_xor(v, o); v = u > v ? u : v; }
    return v;
}
template <typename K>
__device__ __forceinline__ K row_sum(K v, int L) {
    for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// s / (what the renormalisation divides out): see the head of the file; m = 0 keeps s itself
__device__ __forceinline__ float sigmoid_over(float x, float m) {
    return x <= 0.f ? expf(x - m) / (1.f + expf(x)) : 1.f / (1.f + expf(-x));
}

template <typename T, typename K, int V, bool VEC>
__global__ __launch_bounds__(ROUTE_WAVES * kWave) void route_fwd_kernel(RouteArgs a) {
    extern __shared__ float route_lds[];
    int64_t T_ = a.T;
    if (a.n_dev) { const int64_t n = *a.n_dev; T_ = n < T_ ? (n < 0 ? 0 : n) : T_; }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int L = 1 << a.lg_L, Lg = 1 << a.lg_Lg, rpw = kWave >> a.lg_L;
    const int sub = lane & (L - 1), r = lane >> a.lg_L;
    const int64_t t0 = ((int64_t)blockIdx.x * ROUTE_WAVES + wave) * rpw, t = t0 + r;
    if (t0 >= T_) return;                                      // (a whole wave: no block-wide barrier follows)
    const bool on = t < T_ && (!a.selector || a.selector[t]);
    const int Eg = a.E / a.G, g = sub >> a.lg_Lg, lg = sub & (Lg - 1);
    const int e0 = g * Eg + lg * V;
    const int nv = (on && g < a.G) ? min(max(Eg - lg * V, 0), V) : 0;
    float x[V];
    load_logits<T, V, VEC>(reinterpret_cast<const T*>(a.x) + (on ? t : 0) * a.stride + (nv > 0 ? e0 : 0), nv, x);
    bool odd = false;                                          // a logit that leaves the row without a choice to speak of
#pragma unroll
    for (int i = 0; i < V; ++i) odd |= (x[i] != x[i]) || (!a.sigmoid && x[i] == INFINITY);
    const uint64_t odd_lanes = __ballot(odd);
    const bool bad = ((odd_lanes >> (r << a.lg_L)) & (L == 64 ? ~0ull : ((1ull << L) - 1))) != 0;

    // values to choose by; -inf = not there (or already taken)
    K c[V];
    float xmax = 0.f, Z = 1.f;
    if constexpr (sizeof(K) == 4) {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = bad ? -INFINITY : x[i];
        if (!a.sigmoid && !a.renorm) {
            float m = -INFINITY, z = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
            xmax = row_max(m, L);
#pragma unroll
            for (int i = 0; i < V; ++i) z += x[i] > -INFINITY ? expf(x[i] - xmax) : 0.f;
            Z = row_sum(z, L);
        }
    } else {
        double m = -INFINITY, z = 0.0, s[V];
        if (!a.sigmoid) {
#pragma unroll
            for (int i = 0; i < V; ++i) m = fmax(m, (double)x[i]);
            m = row_max(m, L);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double xi = (double)x[i];
            s[i] = !(x[i] > -INFINITY) ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-xi)) : exp(xi - m);
            z += s[i];
        }
        if (!a.sigmoid) {
            z = row_sum(z, L);
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] /= z;
            xmax = (float)m; Z = (float)z;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double b = (a.bias && i < nv) ? (double)a.bias[e0 + i] : 0.0;
            const double v = s[i] + b;
            c[i] = (!bad && x[i] > -INFINITY && v == v) ? (K)v : (K)-INFINITY;
        }
    }

    if (a.top_groups < a.G) {
        // every lane of a group learns the group's value, then how many groups come before it
        K b1 = (K)-INFINITY, b2 = (K)-INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            b2 = c[i] > b1 ? b1 : (c[i] > b2 ? c[i] : b2);
            b1 = c[i] > b1 ? c[i] : b1;
        }
        for (int o = 1; o < Lg; o <<= 1) {
            const K p1 = __shfl_xor(b1, o), p2 = __shfl_xor(b2, o);
            const K lo = p1 < b1 ? p1 : b1;
            b1 = p1 > b1 ? p1 : b1;
            b2 = p2 > b2 ? p2 : b2;
            b2 = lo > b2 ? lo : b2;
        }
        const K mine = a.group_top == 2 ? b1 + b2 : b1;
        int before = 0;
        for (int h = 0; h < a.G; ++h) {
            const K other = __shfl(mine, (r << a.lg_L) + (h << a.lg_Lg));
            before += (other > mine || (other == mine && h < g)) ? 1 : 0;
        }
        if (before >= a.top_groups)
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = (K)-INFINITY;
    }

    float* chosen_x = route_lds + (size_t)wave * rpw * a.k * 2 + (size_t)r * a.k;
    int32_t* chosen_e = reinterpret_cast<int32_t*>(route_lds + (size_t)wave * rpw * a.k * 2 + (size_t)rpw * a.k) + (size_t)r * a.k;
    for (int j = 0; j < a.k; ++j) {
        K best = (K)-INFINITY;
        int be = 0x7fffffff;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (c[i] > best) { best = c[i]; be = e0 + i; }
        for (int o = 1; o < L; o <<= 1) {
            const K ob = __shfl_xor(best, o);
            const int oe = __shfl_xor(be, o);
            if (ob > best || (ob == best && oe < be)) { best = ob; be = oe; }
        }
        if (sub == 0 && be == 0x7fffffff) chosen_e[j] = -1;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < nv && e0 + i == be) { c[i] = (K)-INFINITY; chosen_x[j] = x[i]; chosen_e[j] = be; }
    }
    wave_lds_fence();
    if (t >= T_) return;
    float m = 0.f, S = 1.f;
    if (a.renorm) {
        m = -INFINITY; S = 0.f;
        for (int j = 0; j < a.k; ++j) if (chosen_e[j] >= 0) m = fmaxf(m, chosen_x[j]);
        if (a.sigmoid) m = fminf(m, 0.f);
        for (int j = 0; j < a.k; ++j)
            if (chosen_e[j] >= 0) S += a.sigmoid ? sigmoid_over(chosen_x[j], m) : expf(chosen_x[j] - m);
    } else if (!a.sigmoid) {
        m = xmax; S = Z;
    }
    for (int j = sub; j < a.k; j += L) {
        int e = chosen_e[j];
        float w = 0.f;
        if (e >= 0) w = a.scale * ((a.sigmoid ? sigmoid_over(chosen_x[j], m) : expf(chosen_x[j] - m)) / S);
        if (!on) e = -1;
        else if (bad) { e = j; w = __builtin_nanf(""); }
        a.w[t * a.k + j] = w;
        a.idx[t * a.k + j] = e;
    }
}

// ---- gradient of the logits ---------------------------------------------------------------------------------------
// With A = sum_i g_i w_i / scale:  renormalised softmax  dx_j = w_j (g_j - A), zero elsewhere (the chosen logits alone set the
// ratios); renormalised sigmoid  dx_j = w_j (1 - s_j) (g_j - A);  sigmoid  dx_j = w_j (1 - s_j) g_j;
// softmax  dx_e = [e chosen] w_e g_e - s_e sum_i g_i w_i.  Only the last one reads whole rows of logits again.
template <typename T, int V, bool VEC>
__global__ __launch_bounds__(256) void route_bwd_kernel(RouteArgs a, const float* __restrict__ dw, T* __restrict__ dx) {
    int64_t T_ = a.T;
    if (a.n_dev) { const int64_t n = *a.n_dev; T_ = n < T_ ? (n < 0 ? 0 : n) : T_; }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int L = 1 << a.lg_L, rpw = kWave >> a.lg_L, sub = lane & (L - 1), r = lane >> a.lg_L;
    const int64_t t0 = ((int64_t)blockIdx.x * ROUTE_WAVES + wave) * rpw, t = t0 + r;
    if (t0 >= T_) return;
    const bool on = t < T_;
    const int64_t tt = on ? t : t0;
    const int e0 = sub * V, nv = min(max(a.E - e0, 0), V);
    const T* xp = reinterpret_cast<const T*>(a.x) + tt * a.stride + (nv > 0 ? e0 : 0);
    float d[V];
#pragma unroll
    for (int i = 0; i < V; ++i) d[i] = 0.f;
    float A = 0.f;
    bool mine = false, any = false;
    for (int j = 0; j < a.k; ++j) {
        const int e = a.idx[tt * a.k + j];
        if (e >= 0) {
            any = true;
            A += dw[tt * a.k + j] * a.w[tt * a.k + j];
            mine |= e >= e0 && e < e0 + nv;
        }
    }
    const bool whole = !a.sigmoid && !a.renorm;
    float x[V];
    if (whole || (a.sigmoid && mine)) load_logits<T, V, VEC>(xp, nv, x);
    if (mine) {
        const float shift = a.renorm ? A / a.scale : 0.f;
        for (int j = 0; j < a.k; ++j) {
            const int e = a.idx[tt * a.k + j];
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < nv && e == e0 + i) {
                    float v = a.w[tt * a.k + j] * (dw[tt * a.k + j] - shift);
                    if (a.sigmoid) v *= 1.f / (1.f + expf(x[i]));
                    d[i] += v;
                }
        }
    }
    if (whole) {
        float m = -INFINITY, z = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
        m = row_max(m, L);
        float s[V];
#pragma unroll
        for (int i = 0; i < V; ++i) { s[i] = x[i] > -INFINITY ? expf(x[i] - m) : (x[i] != x[i] ? x[i] : 0.f); z += s[i]; }
        z = row_sum(z, L);
        if (any)
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] -= s[i] / z * A;
    }
    if (!on || nv == 0) return;
    T* out = dx + t * (int64_t)a.E + e0;
    if (VEC) {
        struct alignas(sizeof(T) * V) Pack { T v[V]; } q;
#pragma unroll
        for (int i = 0; i < V; ++i) q.v[i] = (T)d[i];
        *reinterpret_cast<Pack*>(out) = q;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (i < nv) out[i] = (T)d[i];
    }
}

// ---- plan: a stable counting sort of the entries by expert ------------------------------------------------------------
// Entry i = row * top_k + choice.  An entry whose expert is not in [0, E), or whose row lies behind the device-side count, is
// in no segment: its position is -1.  Blocks own consecutive stretches of entries, the waves of a block consecutive parts of
// them; what a wave counts in order lands in order, so equal inputs give equal plans.
constexpr int PLAN_THREADS = 256, PLAN_WAVES = PLAN_THREADS / kWave, PLAN_MAX_E = 512, PLAN_MAX_BLOCKS = 256;

__device__ __forceinline__ int plan_expert(const int32_t* __restrict__ experts, int i, int end, int E) {
    if (i >= end) return -1;
    const int e = experts[i];
    return (e >= 0 && e < E) ? e : -1;
}

__global__ __launch_bounds__(PLAN_THREADS) void plan_count_kernel(const int32_t* __restrict__ experts, int n, int k, int E, int per_block,
                                                                  int32_t* __restrict__ counts, const int64_t* __restrict__ n_dev) {
    __shared__ int32_t hist[PLAN_MAX_E];
    for (int e = threadIdx.x; e < E; e += PLAN_THREADS) hist[e] = 0;
    __syncthreads();
    int end = n;
    if (n_dev) { const int64_t m = *n_dev * k; end = m < n ? (m < 0 ? 0 : (int)m) : n; }
    const int a = blockIdx.x * per_block, b = min(a + per_block, n);
    for (int i = a + threadIdx.x; i < b; i += PLAN_THREADS) {
        const int e = plan_expert(experts, i, end, E);
        if (e >= 0) atomicAdd(&hist[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += PLAN_THREADS) counts[(int64_t)blockIdx.x * E + e] = hist[e];
}

__global__ __launch_bounds__(PLAN_THREADS) void plan_place_kernel(const int32_t* __restrict__ experts, int n, int k, int E, int per_block,
                                                                  const int32_t* __restrict__ counts, int32_t* __restrict__ offsets,
                                                                  int32_t* __restrict__ rows, int32_t* __restrict__ positions,
                                                                  const int64_t* __restrict__ n_dev) {
    __shared__ int32_t cursor[PLAN_WAVES][PLAN_MAX_E];     // next free place of the wave's part, per expert
    __shared__ int32_t base[PLAN_MAX_E];
    __shared__ int32_t wave_total[PLAN_WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, blocks = gridDim.x;
    int end = n;
    if (n_dev) { const int64_t m = *n_dev * k; end = m < n ? (m < 0 ? 0 : (int)m) : n; }
    for (int e = threadIdx.x; e < PLAN_WAVES * PLAN_MAX_E; e += PLAN_THREADS) (&cursor[0][0])[e] = 0;
    __syncthreads();
    // this wave's part
    const int a0 = blockIdx.x * per_block, b0 = min(a0 + per_block, n);
    const int part = per_block / PLAN_WAVES;
    const int a = min(a0 + wave * part, b0), b = min(a + part, b0);
    for (int i = a + lane; i < b; i += kWave) {
        const int e = plan_expert(experts, i, end, E);
        if (e >= 0) atomicAdd(&cursor[wave][e], 1);
    }
    // segment starts (exclusive sum over the experts of all blocks' counts) and what earlier blocks put in front
    int total[PLAN_MAX_E / PLAN_THREADS], before[PLAN_MAX_E / PLAN_THREADS], sum = 0;
#pragma unroll
    for (int q = 0; q < PLAN_MAX_E / PLAN_THREADS; ++q) {
        const int e = threadIdx.x * (PLAN_MAX_E / PLAN_THREADS) + q;
        int tot = 0, bef = 0;
        if (e < E)
            for (int h = 0; h < blocks; ++h) {
                const int v = counts[(int64_t)h * E + e];
                tot += v;
                bef += h < (int)blockIdx.x ? v : 0;
            }
        total[q] = tot; before[q] = bef; sum += tot;
    }
    int scan = sum;
    for (int o = 1; o < kWave; o <<= 1) { const int v = __shfl_up(scan, o); if (lane >= o) scan += v; }
    if (lane == 63) wave_total[wave] = scan;
    __syncthreads();
    int start = scan - sum, all = 0;
    for (int w = 0; w < PLAN_WAVES; ++w) { if (w < wave) start += wave_total[w]; all += wave_total[w]; }
#pragma unroll
    for (int q = 0; q < PLAN_MAX_E / PLAN_THREADS; ++q) {
        const int e = threadIdx.x * (PLAN_MAX_E / PLAN_THREADS) + q;
        if (e < E) {
            base[e] = start + before[q];
            if (blockIdx.x == 0) offsets[e] = start;
            start += total[q];
        }
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[E] = all;
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += PLAN_THREADS) {
        int p = base[e];
        for (int w = 0; w < PLAN_WAVES; ++w) { const int v = cursor[w][e]; cursor[w][e] = p; p += v; }
    }
    __syncthreads();
    for (int i0 = a; i0 < b; i0 += kWave) {
        const int i = i0 + lane;
        const int e = i < b ? plan_expert(experts, i, end, E) : -1;
        uint64_t same = __ballot(e >= 0);
#pragma unroll
        for (int bit = 0; bit < 9; ++bit) {
            const uint64_t m = __ballot((e >> bit) & 1);
            same &= ((e >> bit) & 1) ? m : ~m;
        }
        int place = -1;
        if (e >= 0) place = cursor[wave][e] + __popcll(same & ((1ull << lane) - 1));
        wave_lds_fence();
        if (e >= 0 && (same >> lane) == 1) cursor[wave][e] = place + 1;         // the last one of its expert
        wave_lds_fence();
        if (i < b) positions[i] = place;
        if (place >= 0) rows[place] = i;
    }
    // rows behind the last segment: this block's share of them
    for (int i = max(a0, all) + threadIdx.x; i < b0; i += PLAN_THREADS) rows[i] = -1;
}

// ---- host ---------------------------------------------------------------------------------------------------------
static int lg2_ceil(int v) { int l = 0; while ((1 << l) < v) ++l; return l; }

static int plan_blocks(int64_t n) {
    const int64_t b = (n + 2047) / 2048;
    return (int)(b < 1 ? 1 : b > PLAN_MAX_BLOCKS ? PLAN_MAX_BLOCKS : b);
}

template <typename T, typename K, int V>
static void launch_route_fwd(const RouteArgs& a, bool vec, hipStream_t st) {
    const int rpw = kWave >> a.lg_L;
    const int64_t blocks = (a.T + (int64_t)rpw * ROUTE_WAVES - 1) / ((int64_t)rpw * ROUTE_WAVES);
    const size_t lds = (size_t)ROUTE_WAVES * rpw * a.k * 8;
    if (vec) route_fwd_kernel<T, K, V, true><<<(unsigned)blocks, ROUTE_WAVES * kWave, lds, st>>>(a);
    else route_fwd_kernel<T, K, V, false><<<(unsigned)blocks, ROUTE_WAVES * kWave, lds, st>>>(a);
}

template <typename T, int V>
static void launch_route(const RouteArgs& a, bool wide, bool vec, hipStream_t st) {
    if (wide) launch_route_fwd<T, double, V>(a, vec, st);
    else launch_route_fwd<T, float, V>(a, vec, st);
}

template <typename T, int V>
static void launch_route_bwd(const RouteArgs& a, bool vec, const float* dw, void* dx, hipStream_t st) {
    const int rpw = kWave >> a.lg_L;
    const int64_t blocks = (a.T + (int64_t)rpw * ROUTE_WAVES - 1) / ((int64_t)rpw * ROUTE_WAVES);
    if (vec) route_bwd_kernel<T, V, true><<<(unsigned)blocks, 256, 0, st>>>(a, dw, (T*)dx);
    else route_bwd_kernel<T, V, false><<<(unsigned)blocks, 256, 0, st>>>(a, dw, (T*)dx);
}

static int route_check(const char* what, int dtype, int64_t T, int E, int64_t stride, int k) {
    NSX_REQUIRE(dtype >= NSX_DTYPE_F32 && dtype <= NSX_DTYPE_BF16, "%s: unknown dtype %d", what, dtype);
    NSX_REQUIRE(E >= 1 && E <= NSX_MAX_EXPERTS, "%s: n_experts %d not in [1,%d]", what, E, NSX_MAX_EXPERTS);
    NSX_REQUIRE(k >= 1 && k <= E && k <= NSX_MAX_TOP_K, "%s: top_k %d not in [1,%d] or more than the %d experts", what, k, NSX_MAX_TOP_K, E);
    NSX_REQUIRE(T >= 0 && T <= NSX_MAX_EXPERT_ENTRIES / k, "%s: %lld rows of %d choices are too many", what, (long long)T, k);
    NSX_REQUIRE(stride >= E, "%s: row stride %lld below the %d experts", what, (long long)stride, E);
    return NSX_OK;
}

}  // namespace nsx

extern "C" {

int nsx_expert_route_fwd(const void* logits, int dtype, int64_t T, int E, int64_t row_stride, const float* bias,
                         const uint8_t* selector, int top_k, int sigmoid, int n_groups, int top_groups, int group_top,
                         int renormalise, float scale, float* weights, int32_t* experts, const int64_t* n_device, void* stream) {
    using namespace nsx;
    const int rc = route_check("nsx_expert_route_fwd", dtype, T, E, row_stride, top_k);
    if (rc != NSX_OK) return rc;
    NSX_REQUIRE(n_groups >= 1 && n_groups <= 64 && E % n_groups == 0, "nsx_expert_route_fwd: %d groups of %d experts", n_groups, E);
    NSX_REQUIRE(top_groups >= 1 && top_groups <= n_groups, "nsx_expert_route_fwd: top_groups %d of %d", top_groups, n_groups);
    NSX_REQUIRE(group_top == 1 || group_top == 2, "nsx_expert_route_fwd: group_top %d is not 1 or 2", group_top);
    NSX_REQUIRE(group_top <= E / n_groups, "nsx_expert_route_fwd: group_top %d of groups of %d", group_top, E / n_groups);
    NSX_REQUIRE((int64_t)top_groups * (E / n_groups) >= top_k, "nsx_expert_route_fwd: %d groups of %d experts hold no %d choices",
                top_groups, E / n_groups, top_k);
    NSX_REQUIRE(scale == scale && scale != 0.f, "nsx_expert_route_fwd: scale is 0 or not a number");
    if (T == 0) return NSX_OK;
    NSX_REQUIRE(logits && weights && experts, "nsx_expert_route_fwd: NULL pointer");
    const int Eg = E / n_groups, lg_G = lg2_ceil(n_groups);
    RouteArgs a{logits, row_stride, T, E, bias, selector, top_k, n_groups, top_groups, group_top, sigmoid, renormalise, scale,
                weights, experts, n_device, 0, 0};
    // 16 bytes per lane where the groups are whole numbers of them, else as few values per lane as 64 lanes allow
    int V = dtype == NSX_DTYPE_F32 ? 4 : 8;
    const int esize = dtype == NSX_DTYPE_F32 ? 4 : 2;
    while (V > 4 && Eg % V) V >>= 1;
    while (lg_G + lg2_ceil((Eg + V - 1) / V) > 6) V <<= 1;
    const bool vec = Eg % V == 0 && row_stride % V == 0 && (reinterpret_cast<uintptr_t>(logits) % (size_t)(V * esize)) == 0;
    a.lg_Lg = lg2_ceil((Eg + V - 1) / V);
    a.lg_L = lg_G + a.lg_Lg;
    const bool wide = bias || (top_groups < n_groups && group_top == 2);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype * 32 + V) {
        case 4: launch_route<float, 4>(a, wide, vec, st); break;
        case 8: launch_route<float, 8>(a, wide, vec, st); break;
        case 16: launch_route<float, 16>(a, wide, vec, st); break;
        case 32 + 4: launch_route<half_t, 4>(a, wide, vec, st); break;
        case 32 + 8: launch_route<half_t, 8>(a, wide, vec, st); break;
        case 32 + 16: launch_route<half_t, 16>(a, wide, vec, st); break;
        case 64 + 4: launch_route<bf16_t, 4>(a, wide, vec, st); break;
        case 64 + 8: launch_route<bf16_t, 8>(a, wide, vec, st); break;
        case 64 + 16: launch_route<bf16_t, 16>(a, wide, vec, st); break;
        default: NSX_REQUIRE(false, "nsx_expert_route_fwd: no layout for %d groups of %d experts", n_groups, Eg);
    }
    NSX_LAUNCH_CHECK("nsx_expert_route_fwd");
    return NSX_OK;
}

int nsx_expert_route_bwd(const void* logits, int dtype, int64_t T, int E, int64_t row_stride, int top_k, int sigmoid,
                         int renormalise, float scale, const float* weights, const int32_t* experts, const float* dweights,
                         void* dlogits, const int64_t* n_device, void* stream) {
    using namespace nsx;
    const int rc = route_check("nsx_expert_route_bwd", dtype, T, E, row_stride, top_k);
    if (rc != NSX_OK) return rc;
    if (T == 0) return NSX_OK;
    NSX_REQUIRE(logits && weights && experts && dweights && dlogits, "nsx_expert_route_bwd: NULL pointer");
    RouteArgs a{logits, row_stride, T, E, nullptr, nullptr, top_k, 1, 1, 1, sigmoid, renormalise, scale,
                const_cast<float*>(weights), const_cast<int32_t*>(experts), n_device, 0, 0};
    const int esize = dtype == NSX_DTYPE_F32 ? 4 : 2;
    int V = dtype == NSX_DTYPE_F32 ? (E <= 256 ? 4 : 8) : 8;
    if (dtype != NSX_DTYPE_F32 && E % 8 && E <= 256) V = 4;
    const bool vec = E % V == 0 && row_stride % V == 0 && (reinterpret_cast<uintptr_t>(logits) % (size_t)(V * esize)) == 0 &&
                     (reinterpret_cast<uintptr_t>(dlogits) % (size_t)(V * esize)) == 0;
    a.lg_L = lg2_ceil((E + V - 1) / V);
    hipStream_t st = (hipStream_t)stream;
    switch (dtype * 32 + V) {
        case 4: launch_route_bwd<float, 4>(a, vec, dweights, dlogits, st); break;
        case 8: launch_route_bwd<float, 8>(a, vec, dweights, dlogits, st); break;
        case 32 + 4: launch_route_bwd<half_t, 4>(a, vec, dweights, dlogits, st); break;
        case 32 + 8: launch_route_bwd<half_t, 8>(a, vec, dweights, dlogits, st); break;
        case 64 + 4: launch_route_bwd<bf16_t, 4>(a, vec, dweights, dlogits, st); break;
        default: launch_route_bwd<bf16_t, 8>(a, vec, dweights, dlogits, st); break;
    }
    NSX_LAUNCH_CHECK("nsx_expert_route_bwd");
    return NSX_OK;
}

int64_t nsx_expert_plan_workspace(int64_t n_entries, int E) {
    using namespace nsx;
    NSX_REQUIRE(n_entries >= 0 && n_entries <= NSX_MAX_EXPERT_ENTRIES, "nsx_expert_plan_workspace: %lld entries", (long long)n_entries);
    NSX_REQUIRE(E >= 1 && E <= NSX_MAX_EXPERTS, "nsx_expert_plan_workspace: n_experts %d not in [1,%d]", E, NSX_MAX_EXPERTS);
    return (int64_t)plan_blocks(n_entries) * E * 4;
}

int nsx_expert_plan(const int32_t* experts, int64_t T, int top_k, int E, int32_t* offsets, int32_t* rows, int32_t* positions,
                    void* workspace, const int64_t* n_device, void* stream) {
    using namespace nsx;
    NSX_REQUIRE(E >= 1 && E <= NSX_MAX_EXPERTS, "nsx_expert_plan: n_experts %d not in [1,%d]", E, NSX_MAX_EXPERTS);
    NSX_REQUIRE(top_k >= 1 && top_k <= NSX_MAX_TOP_K, "nsx_expert_plan: top_k %d not in [1,%d]", top_k, NSX_MAX_TOP_K);
    NSX_REQUIRE(T >= 0 && T <= NSX_MAX_EXPERT_ENTRIES / top_k, "nsx_expert_plan: %lld rows of %d choices are too many", (long long)T, top_k);
    NSX_REQUIRE(offsets && workspace, "nsx_expert_plan: NULL pointer");
    const int n = (int)(T * top_k), blocks = plan_blocks(n);
    NSX_REQUIRE(n == 0 || (experts && rows && positions), "nsx_expert_plan: NULL pointer");
    int64_t per = ((int64_t)n + blocks - 1) / blocks;
    per = (per + PLAN_THREADS - 1) / PLAN_THREADS * PLAN_THREADS;
    hipStream_t st = (hipStream_t)stream;
    plan_count_kernel<<<blocks, PLAN_THREADS, 0, st>>>(experts, n, top_k, E, (int)per, (int32_t*)workspace, n_device);
    NSX_LAUNCH_CHECK("nsx_expert_plan");
    plan_place_kernel<<<blocks, PLAN_THREADS, 0, st>>>(experts, n, top_k, E, (int)per, (const int32_t*)workspace, offsets, rows,
                                                       positions, n_device);
    NSX_LAUNCH_CHECK("nsx_expert_plan");
    return NSX_OK;
}

}  // extern "C"
