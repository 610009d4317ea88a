// expert_route.hip -- routed experts: the choice of experts for every row, its gradient, and the plan that orders the
// (row, choice) entries by expert.
//
// Choice.  s_e = softmax(x)_e or 1 / (1 + exp(-x_e)); c_e = s_e + bias_e is what the choice goes by (the bias balances the
// experts' load and has no part in the weights).  With groups, a group counts for the sum of its `group_top` largest c, the
// `top_groups` best groups stay.  The top_k largest c that stay, in falling order, equal values by rising index, are the
// choice; w_j = scale * s_j / sum_i s_i (renormalised) or scale * s_j.
//   * Without a bias (and with groups that count for their largest c) the order of c IS the order of x: the logits are
//     compared as they are and no score is formed for experts that are not chosen.
//   * Otherwise the choice is that of c in 64 bits: two experts whose 32-bit sums round to the same value, or change places,
//     would make it depend on the order of the summation behind the softmax.  c is formed in 32 bits; only where neighbours in
//     the order lie closer than its error are they compared in 64.
//   * Renormalised weights are ratios: of the softmax only exp(x_j - max over the chosen) is left, of the sigmoid
//     exp(x_j - min(max, 0)) / (1 + exp(x_j)) -- neither underflows where all chosen scores are tiny.
// A row is held by L lanes of a wave, V consecutive experts in each (64 / L rows per wave): a row is read once, 16 or 32 bytes
// per lane.  A round of "largest value, lowest index" is log2(L) exchanges of the value within the lanes (DPP), a ballot of the
// lanes that hold it, and the first of them takes its expert out.  The entries lie in LDS, a lane each computes their weights.
// Bound by memory where few are chosen: 2^20 x 32 fp32, top 2: 32 us (151 MB, 4.7 TB/s; a copy reaches 4.96).  By the rounds'
// instructions where many are: 65536 x 256 bf16, top 8: 25 us (38 MB, 1.5 TB/s); with a bias 55 us in fp32; 30011 rows of 8 groups
// 27 us.  (Calls repeated on the same logits, which the caches hold in part: with other data in between the first takes 37, the last 32.
// With all experts of a wave in 64 bits wherever two entries were close the last two took 62 and 35: the few waves that do it end last.)
#include "expert_common.h"
#include <algorithm>

namespace nsx {

struct RouteArgs {
    const void* x; int64_t stride; int64_t T; int E;
    const float* bias; const uint8_t* selector;
    int k, G, top_groups, group_top, sigmoid, renorm; float scale;
    float* w; int32_t* idx; const int64_t* n_dev;
    int lg_L, lg_Lg;                 // lanes per row and per group of it, as powers of two
    FastDiv by_k;
};

constexpr int ROUTE_WAVES = 4;

template <typename T, int V, bool VEC>
__device__ __forceinline__ void load_logits(const T* __restrict__ p, int n, float (&x)[V]) {
    if (VEC) {
        struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack { T v[V]; };
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

// ---- exchanges within the 2^n lanes of a row ----
template <int CTRL> __device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(v, v, CTRL, 0xf, 0xf, false); }
template <int CTRL> __device__ __forceinline__ float dpp(float v) { return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(int, v))); }
template <int CTRL> __device__ __forceinline__ double dpp(double v) {
    const u32x2 b = __builtin_bit_cast(u32x2, v);
    return __builtin_bit_cast(double, u32x2{(uint32_t)dpp<CTRL>((int)b[0]), (uint32_t)dpp<CTRL>((int)b[1])});
}
struct TakeMax { template <typename K> __device__ __forceinline__ K operator()(K a, K b) const { return a > b ? a : b; } };
struct TakeSum { template <typename K> __device__ __forceinline__ K operator()(K a, K b) const { return a + b; } };
// every lane of a row gets the same bits (the operations commute); L is the same for all: the branches are scalar
template <class Op, typename K>
__device__ __forceinline__ K row_all(K v, int L) {
    const Op op;
    if (L > 1) v = op(v, dpp<0xB1>(v));           // quad_perm 1 0 3 2
    if (L > 2) v = op(v, dpp<0x4E>(v));           // quad_perm 2 3 0 1
    if (L > 4) v = op(v, dpp<0x141>(v));          // row_half_mirror: the other quad
    if (L > 8) v = op(v, dpp<0x140>(v));          // row_mirror: the other half of 16
    if (L > 16) v = op(v, __shfl_xor(v, 16));
    if (L > 32) v = op(v, __shfl_xor(v, 32));
    return v;
}
__device__ __forceinline__ uint64_t row_lanes(uint64_t mask, int r, int lg_L) {
    return (mask >> (r << lg_L)) & (lg_L == 6 ? ~0ull : ((1ull << (1 << lg_L)) - 1));
}

// s / (what the renormalisation divides out): see the head of the file; m = 0 keeps s itself
__device__ __forceinline__ float sigmoid_over(float x, float m) {
    return x <= 0.f ? expf(x - m) / (1.f + expf(x)) : 1.f / (1.f + expf(-x));
}

// What is compared: 64-bit values as they are, 32-bit ones as integers of the same order (-0 as 0), whose largest of three is one
// instruction.  Nothing that is compared is NaN.
template <typename K> struct Order;
template <> struct Order<float> {
    typedef int32_t type;
    static __device__ __forceinline__ int32_t of(float v) { const int32_t b = __builtin_bit_cast(int32_t, v + 0.f); return b ^ ((b >> 31) & 0x7fffffff); }
    static __device__ __forceinline__ float value(int32_t k) { return __builtin_bit_cast(float, k ^ ((k >> 31) & 0x7fffffff)); }
    static __device__ __forceinline__ int32_t none() { return 0x807fffff; }                 // of(-inf)
};
template <> struct Order<double> {
    typedef double type;
    static __device__ __forceinline__ double of(double v) { return v; }
    static __device__ __forceinline__ double value(double k) { return k; }
    static __device__ __forceinline__ double none() { return -INFINITY; }
};

// Rounds first .. end of the choice over the wave's rows: an entry of `out` per row each, c of the chosen becomes none.
template <typename K> struct Chosen { K c; int32_t e; };
template <typename K, int V>
__device__ __forceinline__ void choose(const RouteArgs& a, typename Order<K>::type (&c)[V], int e0, int r, int sub, int first, int end, Chosen<K>* __restrict__ out) {
    typedef Order<K> O;
    const int L = 1 << a.lg_L;
    for (int j = first; j < end; ++j) {
        auto best = c[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = c[i] > best ? c[i] : best;
        const auto top = row_all<TakeMax>(best, L);
        const uint64_t holders = row_lanes(__ballot(best == top), r, a.lg_L);
        if (__ffsll((unsigned long long)holders) - 1 == sub) {
            int at = 0;
            bool found = false;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool here = !found && c[i] == top;
                at = here ? i : at;
                c[i] = here ? O::none() : c[i];
                found |= here;
            }
            out[j] = Chosen<K>{O::value(top), top > O::none() ? e0 + at : -1};
        }
    }
    wave_lds_fence();
}

// Distance below which two 32-bit values of the choice may have changed places: twice the error of one.  Sigmoid: the
// exponential is off by (|x| + 2) 2^-23 relatively, which s (1 - s) takes below 3e-7; reciprocal and sums add 2e-7.  Softmax: the
// exponential by |x - max| 2^-24 + 2^-23 relatively, at most 1.5e-7 of 1 after exp(x - max); its sum of up to 512 terms by
// 3e-6 relatively.  Adding the bias rounds once more.
__device__ __forceinline__ float unsure(float v, int sigmoid) { return (sigmoid ? 1e-6f : 8e-6f) + 2.5e-7f * fabsf(v); }

// groups that stay: the values of the others become none.  DOUBT: returns whether the groups are beyond doubt -- each that stays is
// above each that does not by more than their errors.  A group's error is that of its members, which follows their sizes and not that of
// their sum (two large biases may cancel in it), and the sum's rounding.
template <bool DOUBT, typename K, int V>
__device__ __forceinline__ bool keep_groups(const RouteArgs& a, typename Order<K>::type (&c)[V], int r, int g) {
    typedef Order<K> O;
    auto b1 = O::none(), b2 = O::none();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const auto lo = c[i] < b1 ? c[i] : b1;
        b2 = lo > b2 ? lo : b2;
        b1 = c[i] > b1 ? c[i] : b1;
    }
    for (int o = 1; o < 1 << a.lg_Lg; o <<= 1) {
        const auto p1 = __shfl_xor(b1, o), p2 = __shfl_xor(b2, o);
        const auto lo = p1 < b1 ? p1 : b1;
        b1 = p1 > b1 ? p1 : b1;
        b2 = p2 > b2 ? p2 : b2;
        b2 = lo > b2 ? lo : b2;
    }
    // (a group without two experts to choose counts nothing: an infinite bias and none would have no sum)
    const K mine = a.group_top == 2 ? (b2 > O::none() ? O::value(b1) + O::value(b2) : (K)-INFINITY) : O::value(b1);
    int before = 0;
    for (int h = 0; h < a.G; ++h) {
        const K other = __shfl(mine, (r << a.lg_L) + (h << a.lg_Lg));
        before += (other > mine || (other == mine && h < g)) ? 1 : 0;
    }
    const bool stays = before < a.top_groups && g < a.G;
    if (!stays)
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = O::none();
    if constexpr (!DOUBT) return true;
    float off = 0.f;                                           // (infinite sums are what they are)
    if (fabsf(mine) < INFINITY)
        off = 0.5f * unsure(O::value(b1), a.sigmoid) + (a.group_top == 2 ? 0.5f * unsure(O::value(b2), a.sigmoid) + 6e-8f * fabsf(mine) : 0.f);
    const float lowest = -row_all<TakeMax>(stays ? off - mine : -INFINITY, 1 << a.lg_L);
    const float highest = row_all<TakeMax>(stays || g >= a.G ? -INFINITY : mine + off, 1 << a.lg_L);
    return lowest - highest > 0.f;
}

// SCORES: the choice goes by scores, else by the logits themselves.  32 bits first; where neighbours of the choice lie closer than
// `unsure`, the chosen and the one that just missed are compared in 64 bits, where more may have taken part all experts of the rows.
template <typename T, int V, bool VEC, bool SCORES>
__global__ __launch_bounds__(ROUTE_WAVES * kWave) void route_fwd_kernel(RouteArgs a) {
    extern __shared__ __attribute__((aligned(16))) char route_lds[];
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
    const T* row = reinterpret_cast<const T*>(a.x) + (on ? t : 0) * a.stride;
    float x[V];
    load_logits<T, V, VEC>(row + (nv > 0 ? e0 : 0), nv, x);
    bool odd = false;                                          // a logit that leaves the row without a choice to speak of
#pragma unroll
    for (int i = 0; i < V; ++i) odd |= (x[i] != x[i]) || (!a.sigmoid && x[i] == INFINITY);
    const bool bad = row_lanes(__ballot(odd), r, a.lg_L) != 0;

    const int slots = a.k + (SCORES ? 2 : 0);
    char* mine = route_lds + (size_t)(wave * rpw + r) * slots * (SCORES ? sizeof(Chosen<double>) : sizeof(Chosen<float>));
    Chosen<float>* out = reinterpret_cast<Chosen<float>*>(mine);
    float xmax = 0.f, Z = 1.f;                                 // softmax over the whole row, where it is asked for
    if (!a.sigmoid && (SCORES || !a.renorm)) {
        float m = x[0], z = 0.f;
#pragma unroll
        for (int i = 1; i < V; ++i) m = fmaxf(m, x[i]);
        xmax = row_all<TakeMax>(m, L);
#pragma unroll
        for (int i = 0; i < V; ++i) z += x[i] > -INFINITY ? expf(x[i] - xmax) : 0.f;
        Z = row_all<TakeSum>(z, L);
    }
    int32_t c[V];
    bool again = false;
    if (!SCORES) {
#pragma unroll
        for (int i = 0; i < V; ++i) c[i] = bad ? Order<float>::none() : Order<float>::of(x[i]);
        if (a.top_groups < a.G) keep_groups<false, float>(a, c, r, g);
        choose<float>(a, c, e0, r, sub, 0, a.k, out);
    } else {
        float bias[V];
#pragma unroll
        for (int i = 0; i < V; ++i) bias[i] = 0.f;
        if (a.bias) {
            if (VEC) { if (nv > 0) __builtin_memcpy(bias, a.bias + e0, V * sizeof(float)); }
            else {
#pragma unroll
                for (int i = 0; i < V; ++i) if (i < nv) bias[i] = a.bias[e0 + i];
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float s = a.sigmoid ? __builtin_amdgcn_rcpf(1.f + __expf(-x[i])) : expf(x[i] - xmax) * (1.f / Z);
            const float v = s + bias[i];
            c[i] = (!bad && x[i] > -INFINITY && v == v) ? Order<float>::of(v) : Order<float>::none();
        }
        bool whole = false;                                    // the groups that stay, or more than one expert behind the choice, are in doubt
        if (a.top_groups < a.G) whole = !keep_groups<true, float>(a, c, r, g) && !bad;
        choose<float>(a, c, e0, r, sub, 0, a.k + 1, out);
        for (int j = sub; j < a.k; j += L) {
            const Chosen<float> p = out[j], q = out[j + 1];
            // (equal logits and biases are equal in 64 bits as well -- unless a third that is not may come between the last
            // that is chosen and the first that is not)
            if (q.e >= 0 && !(p.c - q.c > unsure(p.c, a.sigmoid)))
                again |= j == a.k - 1 || !((float)row[p.e] == (float)row[q.e] && (!a.bias || a.bias[p.e] == a.bias[q.e]));
        }
        wave_lds_fence();
        if (__ballot((again || whole) && on) != 0) {
            choose<float>(a, c, e0, r, sub, a.k + 1, a.k + 2, out);
            const Chosen<float> last = out[a.k - 1], third = out[a.k + 1];
            whole |= third.e >= 0 && !(last.c - third.c > unsure(last.c, a.sigmoid));
            const bool all = __ballot(whole && on) != 0;
            double d[V], m = -INFINITY, z = 0.0;
            if (all || !a.sigmoid) {
                if (!a.sigmoid) {
#pragma unroll
                    for (int i = 0; i < V; ++i) m = fmax(m, (double)x[i]);
                    m = row_all<TakeMax>(m, L);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const double xi = (double)x[i];
                    d[i] = !(x[i] > -INFINITY) ? 0.0 : a.sigmoid ? 1.0 / (1.0 + exp(-xi)) : exp(xi - m);
                    z += d[i];
                }
                if (!a.sigmoid) z = row_all<TakeSum>(z, L);
            }
            if (all) {
                Chosen<double>* wide = reinterpret_cast<Chosen<double>*>(mine);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const double v = (a.sigmoid ? d[i] : d[i] / z) + (double)bias[i];
                    d[i] = (!bad && x[i] > -INFINITY && v == v) ? v : -INFINITY;
                }
                if (a.top_groups < a.G) keep_groups<false, double>(a, d, r, g);
                choose<double>(a, d, e0, r, sub, 0, a.k, wide);
                // (back to the narrow entries; a row's first lane moves them in order: entry j lies in front of what it comes from.  Byte by
                // byte for the compiler, which may take a store of one type for no business of a load of another.)
                if (sub == 0)
                    for (int j = 0; j < a.k; ++j) {
                        Chosen<double> w;
                        __builtin_memcpy(&w, wide + j, sizeof w);
                        const Chosen<float> narrow{(float)w.c, w.e};
                        __builtin_memcpy(out + j, &narrow, sizeof narrow);
                    }
            } else {
                // The k + 1 candidates in 64 bits, an entry to a lane, then by their rank.
                double* v = reinterpret_cast<double*>(mine + slots * sizeof(Chosen<float>));
                int32_t* sorted = reinterpret_cast<int32_t*>(v);
                for (int j = sub; j <= a.k; j += L) {
                    const int e = out[j].e;
                    const double xe = e >= 0 ? (double)(float)row[e] : 0.0;
                    v[j] = e < 0 ? -INFINITY : (a.sigmoid ? 1.0 / (1.0 + exp(-xe)) : exp(xe - m) / z) + (a.bias ? (double)a.bias[e] : 0.0);
                }
                wave_lds_fence();
                for (int j = sub; j <= a.k; j += L) {
                    const int e = out[j].e;
                    const double own = v[j];
                    int rank = 0;
                    for (int i = 0; i <= a.k; ++i) {
                        const int f = out[i].e;
                        const double other = v[i];
                        rank += other > own || (other == own && (f < 0 || e < 0 ? i < j : f < e)) ? 1 : 0;
                    }
                    out[j].c = __builtin_bit_cast(float, rank);
                }
                wave_lds_fence();
                for (int j = sub; j <= a.k; j += L) sorted[__builtin_bit_cast(int, out[j].c)] = out[j].e;
                wave_lds_fence();
                for (int j = sub; j < a.k; j += L) out[j].e = sorted[j];
            }
            wave_lds_fence();
        }
    }
    // the weights: an entry to a lane, which keeps its logit in c's place
    float m = -INFINITY, S = 0.f;
    for (int j = sub; j < a.k; j += L) {
        const float v = out[j].e >= 0 ? (float)row[out[j].e] : -INFINITY;
        out[j].c = v;
        m = fmaxf(m, v);
    }
    if (a.renorm) {
        m = row_all<TakeMax>(m, L);
        if (a.sigmoid) m = fminf(m, 0.f);
        for (int j = sub; j < a.k; j += L)
            if (out[j].e >= 0) S += a.sigmoid ? sigmoid_over(out[j].c, m) : expf(out[j].c - m);
        S = row_all<TakeSum>(S, L);
    } else {
        m = a.sigmoid ? 0.f : xmax;
        S = Z;
    }
    if (t >= T_) return;
    for (int j = sub; j < a.k; j += L) {
        int e = out[j].e;
        float w = 0.f;
        if (e >= 0) w = a.scale * ((a.sigmoid ? sigmoid_over(out[j].c, m) : expf(out[j].c - m)) / S);
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
// A wave's rows lie in LDS as 32-bit values: cleared, the chosen places written by one lane per entry, read back and stored
// whole -- the entries are read once and no lane compares its experts with them.
// Bound by memory: 2^20 x 32 fp32, top 2 renormalised: 26 us for 159 MB (the caches take part of them; a copy: 32); the whole
// softmax, which reads the logits as well, 68 for 293 (59).  fp32 rows leave 16 bytes per lane side by side (32 per lane: 29 us).
// Stores past the caches (nontemporal) took 21 us, but what they gain the next reader of the gradient pays: together 81 | 82 us.
template <typename T, int V, bool VEC>
__global__ __launch_bounds__(256) void route_bwd_kernel(RouteArgs a, const float* __restrict__ dw, T* __restrict__ dx) {
    extern __shared__ __attribute__((aligned(16))) char route_lds[];
    int64_t T_ = a.T;
    if (a.n_dev) { const int64_t n = *a.n_dev; T_ = n < T_ ? (n < 0 ? 0 : n) : T_; }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int L = 1 << a.lg_L, rpw = kWave >> a.lg_L, sub = lane & (L - 1), r = lane >> a.lg_L;
    const int64_t t0 = ((int64_t)blockIdx.x * ROUTE_WAVES + wave) * rpw, t = t0 + r;
    if (t0 >= T_) return;
    const int rows = (int)min((int64_t)rpw, T_ - t0), e0 = sub * V, nv = r < rows ? min(max(a.E - e0, 0), V) : 0;
    const bool whole = !a.sigmoid && !a.renorm;
    float* d = reinterpret_cast<float*>(route_lds) + (size_t)wave * (64 * V + ((rpw * a.k + 3) & ~3));   // [rpw][L * V]
    float* gw = d + 64 * V;                                                                     // [rpw][k]
    f32x4* own = reinterpret_cast<f32x4*>(d + lane * V);
    float x[V];
    if (whole) load_logits<T, V, VEC>(reinterpret_cast<const T*>(a.x) + (r < rows ? t : t0) * a.stride + (nv > 0 ? e0 : 0), nv, x);
#pragma unroll
    for (int i = 0; i < V / 4; ++i) own[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int n = rows * a.k;
    for (int i = lane; i < n; i += kWave) {
        const int64_t at = t0 * a.k + i;
        gw[i] = a.idx[at] >= 0 ? dw[at] * a.w[at] : 0.f;
    }
    wave_lds_fence();
    for (int i = lane; i < n; i += kWave) {
        const int64_t at = t0 * a.k + i;
        const int row = a.by_k(i), e = a.idx[at];
        float v = gw[i];
        if (a.renorm) {
            float A = 0.f;
            for (int j = 0; j < a.k; ++j) A += gw[row * a.k + j];
            v -= a.w[at] * (A / a.scale);
        }
        if ((unsigned)e < (unsigned)a.E) {
            if (a.sigmoid) v *= 1.f / (1.f + expf((float)reinterpret_cast<const T*>(a.x)[(t0 + row) * a.stride + e]));
            d[row * (L * V) + e] = v;
        }
    }
    wave_lds_fence();
    float o[V];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        const f32x4 v = own[i];
#pragma unroll
        for (int q = 0; q < 4; ++q) o[i * 4 + q] = v[q];
    }
    if (whole) {
        float m = x[0], z = 0.f, s[V], A = 0.f;
#pragma unroll
        for (int i = 1; i < V; ++i) m = fmaxf(m, x[i]);
        m = row_all<TakeMax>(m, L);
#pragma unroll
        for (int i = 0; i < V; ++i) { s[i] = x[i] > -INFINITY ? expf(x[i] - m) : (x[i] != x[i] ? x[i] : 0.f); z += s[i]; }
        z = row_all<TakeSum>(z, L);
        bool any = false;
        if (r < rows)
            for (int j = 0; j < a.k; ++j) { A += gw[r * a.k + j]; any |= a.idx[t * a.k + j] >= 0; }
        if (any)
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] -= s[i] / z * A;
    }
    if (sizeof(T) == 4 && VEC && a.E == L * V) {               // the wave's rows are one stretch of memory: 16 bytes per lane, side by side
        if (whole) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) own[i] = f32x4{o[i * 4], o[i * 4 + 1], o[i * 4 + 2], o[i * 4 + 3]};
            wave_lds_fence();
        }
        for (int i = lane * 4; i < rows * a.E; i += kWave * 4)
            *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(dx) + t0 * (int64_t)a.E + i) = *reinterpret_cast<const f32x4*>(d + i);
        return;
    }
    if (nv == 0) return;
    T* p = dx + t * (int64_t)a.E + e0;
    if (VEC) {
        struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack { T v[V]; } q;
#pragma unroll
        for (int i = 0; i < V; ++i) q.v[i] = (T)o[i];
        *reinterpret_cast<Pack*>(p) = q;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) if (i < nv) p[i] = (T)o[i];
    }
}

// ---- plan: a stable counting sort of the entries by expert ------------------------------------------------------------
// Entry i = row * top_k + choice.  An entry whose expert is not in [0, E), or whose row lies behind the device-side count, is
// in no segment: its position is -1.  Blocks own consecutive stretches of entries, the waves of a block consecutive parts of
// them; what a wave counts in order lands in order, so equal inputs give equal plans.  A first launch counts every block's entries
// per expert; in the second a block knows from all counts where its own begin, and places them 64 at a time: lanes of one expert
// find each other by ballots of the expert's bits.
// Bound by the chain of steps: 2^20 rows x 2 of 16 experts, 25 MB: 16.6 us, 1.5 TB/s (a copy would take 5); 4096 x 2: 7.7 us, of
// which one launch is 3.  8 entries per lane are loaded ahead; one at a time took 111 us.
constexpr int PLAN_MAX_BLOCKS = 256;
constexpr int PLAN_LANE = 8, PLAN_PIECE = PLAN_LANE * kWave;      // entries that a lane, a wave loads at a time

__device__ __forceinline__ void plan_load(const int32_t* __restrict__ experts, int i0, int end, int E, int (&e)[PLAN_LANE]) {
#pragma unroll
    for (int q = 0; q < PLAN_LANE; ++q) {
        const int i = i0 + q * kWave + (threadIdx.x & 63);
        e[q] = i < end ? experts[i] : -1;
    }
#pragma unroll
    for (int q = 0; q < PLAN_LANE; ++q) e[q] = (unsigned)e[q] < (unsigned)E ? e[q] : -1;
}
__device__ __forceinline__ int plan_end(int n, int k, const int64_t* __restrict__ n_dev) {
    if (!n_dev) return n;
    const int64_t m = *n_dev;
    return m < 0 ? 0 : (m < n / k ? (int)m * k : n);
}

// entries per expert of each block
template <int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void plan_count_kernel(const int32_t* __restrict__ experts, int n, int k, int E, int per_block,
                                                                  int32_t* __restrict__ counts, const int64_t* __restrict__ n_dev) {
    constexpr int PLAN_THREADS = WAVES * kWave;
    __shared__ int32_t hist[NSX_MAX_EXPERTS];
    for (int e = threadIdx.x; e < E; e += PLAN_THREADS) hist[e] = 0;
    __syncthreads();
    const int wave = threadIdx.x >> 6, a = blockIdx.x * per_block, b = min(a + per_block, plan_end(n, k, n_dev));
    for (int i = a + wave * PLAN_PIECE; i < b; i += WAVES * PLAN_PIECE) {
        int e[PLAN_LANE];
        plan_load(experts, i, b, E, e);
#pragma unroll
        for (int q = 0; q < PLAN_LANE; ++q) if (e[q] >= 0) atomicAdd(&hist[e[q]], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += PLAN_THREADS) counts[(int64_t)blockIdx.x * E + e] = hist[e];
}

// bits: of an expert's number; 1 << bits <= the threads: the blocks' counts are summed column by column, several threads to a column
template <int WAVES>
__global__ __launch_bounds__(WAVES * kWave) void plan_place_kernel(const int32_t* __restrict__ experts, int n, int k, int E, int bits, int per_block,
                                                                  const int32_t* __restrict__ counts, int32_t* __restrict__ offsets,
                                                                  int32_t* __restrict__ rows, int32_t* __restrict__ positions,
                                                                  const int64_t* __restrict__ n_dev) {
    constexpr int PLAN_THREADS = WAVES * kWave, MAX_E = WAVES == 16 ? NSX_MAX_EXPERTS : WAVES == 8 ? 256 : 32;
    __shared__ int32_t cursor[WAVES][MAX_E];                    // next free place of the wave's part, per expert
    __shared__ int32_t part_all[PLAN_THREADS], part_before[PLAN_THREADS];
    __shared__ int32_t all[MAX_E], first[MAX_E];
    __shared__ int32_t routed;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, blocks = gridDim.x;
    const int end = plan_end(n, k, n_dev);
    for (int x = lane; x < E; x += kWave) cursor[wave][x] = 0;
    __syncthreads();
    const int a0 = blockIdx.x * per_block, b0 = min(a0 + per_block, n), part = per_block / WAVES;
    const int a = min(a0 + wave * part, b0), b = min(a + part, b0), live = min(b, end);
    int e[PLAN_LANE];
    for (int i = a; i < live; i += PLAN_PIECE) {
        plan_load(experts, i, live, E, e);
#pragma unroll
        for (int q = 0; q < PLAN_LANE; ++q) if (e[q] >= 0) atomicAdd(&cursor[wave][e[q]], 1);
    }
    // of every expert: all entries, and those of earlier blocks
    if (blocks > 1) {
        const int col = threadIdx.x & ((1 << bits) - 1), parts = PLAN_THREADS >> bits;
        int sum = 0, before = 0;
        if (col < E) {
#pragma unroll 8
            for (int h = threadIdx.x >> bits; h < blocks; h += parts) {
                const int v = counts[(int64_t)h * E + col];
                sum += v;
                before += h < (int)blockIdx.x ? v : 0;
            }
        }
        part_all[threadIdx.x] = sum;
        part_before[threadIdx.x] = before;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < E; x += PLAN_THREADS) {
        int sum = 0, before = 0;
        if (blocks > 1) {
#pragma unroll 4
            for (int h = x; h < PLAN_THREADS; h += 1 << bits) { sum += part_all[h]; before += part_before[h]; }
        } else {
#pragma unroll
            for (int w = 0; w < WAVES; ++w) sum += cursor[w][x];
        }
        all[x] = sum;
        first[x] = before;
    }
    __syncthreads();
    if (wave == 0) {
        constexpr int PER = NSX_MAX_EXPERTS / kWave;
        int sum = 0;
#pragma unroll
        for (int q = 0; q < PER; ++q) { const int x = lane * PER + q; if (x < E) sum += all[x]; }
        int scan = sum;
        for (int o = 1; o < kWave; o <<= 1) { const int v = __shfl_up(scan, o); if (lane >= o) scan += v; }
        int start = scan - sum;
#pragma unroll
        for (int q = 0; q < PER; ++q) {
            const int x = lane * PER + q;
            if (x < E) {
                first[x] += start;
                if (blockIdx.x == 0) offsets[x] = start;
                start += all[x];
            }
        }
        if (lane == 63) {
            routed = scan;
            if (blockIdx.x == 0) offsets[E] = scan;
        }
    }
    __syncthreads();
    for (int x = threadIdx.x; x < E; x += PLAN_THREADS) {
        int p = first[x], v[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v[w] = cursor[w][x];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) { cursor[w][x] = p; p += v[w]; }
    }
    __syncthreads();
    const bool kept = b - a <= PLAN_PIECE;                        // (the entries are still in registers)
    for (int i0 = a; i0 < b; i0 += PLAN_PIECE) {
        if (!kept || i0 >= live) plan_load(experts, i0, live, E, e);
#pragma unroll
        for (int q = 0; q < PLAN_LANE; ++q) {
            const int i = i0 + q * kWave + lane;
            // lanes with the same expert, by its bits; the lowest free place, then one more for each of them
            uint64_t same = __ballot(e[q] >= 0);
            for (int bit = 0; bit < bits; ++bit) {
                const bool set = (e[q] >> bit) & 1;
                const uint64_t m = __ballot(set);
                same &= set ? m : ~m;
            }
            int place = -1;
            if (e[q] >= 0) place = cursor[wave][e[q]] + __popcll(same & ((1ull << lane) - 1));
            wave_lds_fence();
            if (e[q] >= 0 && (same >> lane) == 1) cursor[wave][e[q]] = place + 1;         // the last of them
            wave_lds_fence();
            if (i < b) positions[i] = place;
            if (place >= 0) rows[place] = i;
        }
    }
    // rows behind the last segment: this block's share of them
    for (int i = max(a0, routed) + threadIdx.x; i < b0; i += PLAN_THREADS) rows[i] = -1;
}

// ---- host ---------------------------------------------------------------------------------------------------------
static int lg2_ceil(int v) { int l = 0; while ((1 << l) < v) ++l; return l; }

// Waves per block: one launch of 16 does up to 8192 entries; of more, short blocks spread the work over the CUs while every block
// reads every other's counts.  us with 4 | 8 | 16:  524288 entries of 16 experts  10.9 | 12.5 | 14.9;  of 64  13.1 | 11.7 | 13.9;
// of 256  23.9 | 14.8 | 15.0;  131072 of 256  13.2 | 11.8 | 14.1;  2^20 of 64  19.1 | 13.8 | 15.2;  2^21 of 16  24.0 | 18.5 | 18.4
static int plan_waves(int64_t n, int E) {
    if (n <= 16 * PLAN_PIECE || E > 256 || n > PLAN_MAX_BLOCKS * 8 * PLAN_PIECE) return 16;
    return E <= 32 && n <= PLAN_MAX_BLOCKS * 4 * PLAN_PIECE ? 4 : 8;
}
static int plan_blocks(int64_t n, int E) {
    const int64_t piece = (int64_t)plan_waves(n, E) * PLAN_PIECE, b = (n + piece - 1) / piece;
    return (int)(b < 1 ? 1 : b > PLAN_MAX_BLOCKS ? PLAN_MAX_BLOCKS : b);
}

template <int WAVES>
static void launch_plan(int blocks, const int32_t* experts, int n, int k, int E, int per, int32_t* counts, int32_t* offsets, int32_t* rows,
                        int32_t* positions, const int64_t* n_dev, hipStream_t st) {
    if (blocks > 1) plan_count_kernel<WAVES><<<blocks, WAVES * kWave, 0, st>>>(experts, n, k, E, per, counts, n_dev);
    plan_place_kernel<WAVES><<<blocks, WAVES * kWave, 0, st>>>(experts, n, k, E, lg2_ceil(E), per, counts, offsets, rows, positions, n_dev);
}

// bytes of LDS that a workgroup's entries take
static size_t route_lds_bytes(int lg_L, int k, bool by_scores) {
    return (size_t)ROUTE_WAVES * (kWave >> lg_L) * (by_scores ? (k + 2) * sizeof(Chosen<double>) : k * sizeof(Chosen<float>));
}

template <typename T, int V>
static void launch_route(const RouteArgs& a, bool by_scores, bool vec, hipStream_t st) {
    const int rpw = kWave >> a.lg_L;
    const unsigned blocks = (unsigned)((a.T + (int64_t)rpw * ROUTE_WAVES - 1) / ((int64_t)rpw * ROUTE_WAVES));
    const size_t lds = route_lds_bytes(a.lg_L, a.k, by_scores);
    if (by_scores) {
        if (vec) route_fwd_kernel<T, V, true, true><<<blocks, ROUTE_WAVES * kWave, lds, st>>>(a);
        else route_fwd_kernel<T, V, false, true><<<blocks, ROUTE_WAVES * kWave, lds, st>>>(a);
    } else {
        if (vec) route_fwd_kernel<T, V, true, false><<<blocks, ROUTE_WAVES * kWave, lds, st>>>(a);
        else route_fwd_kernel<T, V, false, false><<<blocks, ROUTE_WAVES * kWave, lds, st>>>(a);
    }
}

template <typename T, int V>
static void launch_route_bwd(const RouteArgs& a, bool vec, const float* dw, void* dx, hipStream_t st) {
    const int rpw = kWave >> a.lg_L;
    const unsigned blocks = (unsigned)((a.T + (int64_t)rpw * ROUTE_WAVES - 1) / ((int64_t)rpw * ROUTE_WAVES));
    const size_t lds = (size_t)ROUTE_WAVES * (64 * V + ((rpw * a.k + 3) & ~3)) * 4;
    if (vec) route_bwd_kernel<T, V, true><<<blocks, ROUTE_WAVES * kWave, lds, st>>>(a, dw, (T*)dx);
    else route_bwd_kernel<T, V, false><<<blocks, ROUTE_WAVES * kWave, lds, st>>>(a, dw, (T*)dx);
}

// rows of logits can be read (and written) V at a time
static bool route_vec(const void* p, int V, int esize, int64_t stride, int group) {
    const size_t align = std::min<size_t>(16, (size_t)V * esize);
    return group % V == 0 && (size_t)stride * esize % align == 0 && reinterpret_cast<uintptr_t>(p) % align == 0;
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
                weights, experts, n_device, 0, 0, fast_div(top_k)};
    // Values per lane: 16 leave the fewest exchanges and instructions per row, 4 the shortest chain where few waves hide it.  us with
    // 4 | 8 | 16 (groups: 8 with a bias, the best 2 of each counting, 4 of them stay):
    //   2^20 x 32 fp32 top 2      62 | 38 | 32     16384 x 64 fp32 top 6           6.0 |  5.5 |  6.8    30011 x 256 bf16 top 8, groups  48 | 31 | 27
    //   65536 x 256 bf16 top 8    58 | 35 | 25      4096 x 64 fp32 top 6           4.5 |  5.0 |  6.7     2^20 x 8 fp16 top 2            17 | 13 | 13
    //   2^18 x 64 fp32 top 6      46 | 33 | 30      4096 x 256 bf16 top 8, groups 14.7 | 15.7 | 20.2     1 x 64 fp32 top 6             4.5 | 4.3 | 5.7
    int V = T * E <= 1 << 19 ? 4 : T * E <= 1 << 22 || Eg < 32 ? 8 : 16;
    const int esize = dtype == NSX_DTYPE_F32 ? 4 : 2;
    while (V > 4 && Eg % V) V >>= 1;
    while (lg_G + lg2_ceil((Eg + V - 1) / V) > 6) V <<= 1;
    const bool wide = bias || (top_groups < n_groups && group_top == 2);
    // (rows of few lanes and many choices: more lanes per row where a workgroup's entries would pass 64 KB)
    while (V > 4 && route_lds_bytes(lg_G + lg2_ceil((Eg + V - 1) / V), top_k, wide) > 65536) V >>= 1;
    const bool vec = route_vec(logits, V, esize, row_stride, Eg);
    a.lg_Lg = lg2_ceil((Eg + V - 1) / V);
    a.lg_L = lg_G + a.lg_Lg;
    NSX_REQUIRE(a.lg_L <= 6 && route_lds_bytes(a.lg_L, top_k, wide) <= 65536, "nsx_expert_route_fwd: no layout for %d choices of %d groups of %d experts",
                top_k, n_groups, Eg);
    NSX_REQUIRE((T << a.lg_L) + 256 < ((int64_t)1 << 32), "nsx_expert_route_fwd: %lld rows of %d lanes are more than one launch",
                (long long)T, 1 << a.lg_L);
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
                const_cast<float*>(weights), const_cast<int32_t*>(experts), n_device, 0, 0, fast_div(top_k)};
    const int esize = dtype == NSX_DTYPE_F32 ? 4 : 2;
    const int V = E % 8 && E <= 256 ? 4 : 8;
    const bool vec = route_vec(logits, V, esize, row_stride, E) && route_vec(dlogits, V, esize, E, E);
    a.lg_L = lg2_ceil((E + V - 1) / V);
    NSX_REQUIRE((T << a.lg_L) + 256 < ((int64_t)1 << 32), "nsx_expert_route_bwd: %lld rows of %d lanes are more than one launch",
                (long long)T, 1 << a.lg_L);
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
    return (int64_t)plan_blocks(n_entries, E) * E * 4;
}

int nsx_expert_plan(const int32_t* experts, int64_t T, int top_k, int E, int32_t* offsets, int32_t* rows, int32_t* positions,
                    void* workspace, const int64_t* n_device, void* stream) {
    using namespace nsx;
    NSX_REQUIRE(E >= 1 && E <= NSX_MAX_EXPERTS, "nsx_expert_plan: n_experts %d not in [1,%d]", E, NSX_MAX_EXPERTS);
    NSX_REQUIRE(top_k >= 1 && top_k <= NSX_MAX_TOP_K, "nsx_expert_plan: top_k %d not in [1,%d]", top_k, NSX_MAX_TOP_K);
    NSX_REQUIRE(T >= 0 && T <= NSX_MAX_EXPERT_ENTRIES / top_k, "nsx_expert_plan: %lld rows of %d choices are too many", (long long)T, top_k);
    NSX_REQUIRE(offsets && workspace, "nsx_expert_plan: NULL pointer");
    const int n = (int)(T * top_k), waves = plan_waves(n, E), blocks = plan_blocks(n, E);
    NSX_REQUIRE(n == 0 || (experts && rows && positions), "nsx_expert_plan: NULL pointer");
    const int64_t piece = (int64_t)waves * PLAN_PIECE, per = (((int64_t)n + blocks - 1) / blocks + piece - 1) / piece * piece;
    hipStream_t st = (hipStream_t)stream;
    int32_t* counts = (int32_t*)workspace;
    if (waves == 16) launch_plan<16>(blocks, experts, n, top_k, E, (int)per, counts, offsets, rows, positions, n_device, st);
    else if (waves == 8) launch_plan<8>(blocks, experts, n, top_k, E, (int)per, counts, offsets, rows, positions, n_device, st);
    else launch_plan<4>(blocks, experts, n, top_k, E, (int)per, counts, offsets, rows, positions, n_device, st);
    NSX_LAUNCH_CHECK("nsx_expert_plan");
    return NSX_OK;
}

}  // extern "C"
