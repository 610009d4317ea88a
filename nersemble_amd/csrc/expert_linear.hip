// expert_linear.hip -- routed experts: every ordered row times the weight matrix of its expert, and the two gradients.
//
//   y_p = act(W_e x_r(p)),   dx_p = W_e^T dz_p,   dW_e = sum_{p in e} dz_p x_r(p)^T,   dz = dy where y > 0 (ReLU) or dy
//
// All three are D[m][c] = sum_q P[m][q] Q[c][q] with m the index that is contiguous in memory in the result:
//   forward  m = output feature, c = ordered row,      q = input feature    P = W (q contiguous)  Q = x (q contiguous)
//   dx       m = input feature,  c = ordered row,      q = output feature   P = W (m contiguous)  Q = dz (q contiguous)
//   dW       m = input feature,  c = output feature,   q = ordered row      P = x (m contiguous)  Q = dz (c contiguous)
// One kernel: 16-bit tiles of P and Q in LDS with q contiguous (128 B per row, 16-byte pieces permuted by the row's number so
// that neither the stores nor the fragment reads of 16 rows share banks), v_mfma_f32_16x16x32, 32-bit accumulators.  What is
// not q-contiguous in memory is turned on its way through the registers: 4 q x 8 m per thread, 16 byte permutations, eight
// 8-byte stores.  A lane holds 4 consecutive m of one c: 8-byte (16-byte for 32-bit gradients) stores.
// Segments are read from the plan on the device: the grid covers the most tiles that any split of R rows over E experts can
// have, every workgroup finds its (expert, tile) by one scan of the offsets.
#include "expert_common.h"

namespace nsx {

enum LinMode { LIN_FWD, LIN_DX, LIN_DW };

struct LinArgs {
    const void *p, *q, *mask;        // mask: y (16-bit), dz = 0 where it is 0; laid out as q
    void* d;
    int64_t ldp, ldq, ldmask, ldd;   // elements
    int64_t p_expert, d_expert;      // elements from one expert's matrix to the next
    const int32_t *offsets, *rows;   // rows: NULL = x holds ordered rows
    FastDiv top_k;
    int E, R, x_rows;
    int M, C, K;                     // extents of m, c (dW) and q (forward, dx)
    int m_tiles, c_tiles, splits, relu;
    float* partial;                  // dW with splits > 1: [split][E][C][M]
};

template <typename T> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma16<half_t>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Elem<half_t>::x8, a), __builtin_bit_cast(Elem<half_t>::x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<bf16_t>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Elem<bf16_t>::x8, a), __builtin_bit_cast(Elem<bf16_t>::x8, b), c, 0, 0, 0);
}

constexpr int LIN_BQ = 64;           // q per step: 128 B of 16-bit values
__device__ __forceinline__ uint32_t lds_piece(int row, int ch) { return (uint32_t)(row * 128 + ((ch ^ (row ^ (row >> 3))) & 7) * 16); }

// both 16-bit halves of `v` kept where those of `y` (not negative) are not zero
__device__ __forceinline__ uint32_t keep_where(uint32_t v, uint32_t y) {
    const uint32_t t = ((y & 0x7fff7fffu) + 0x7fff7fffu) & 0x80008000u;
    return v & (t | (t - (t >> 15)));
}

// One operand's share of a thread: ROWS rows (of m or c) x 64 q per step, by NT threads.
template <int ROWS, int NT, bool MASK>
struct AlongQ {                      // q contiguous in memory
    static constexpr int N = ROWS * 8 / NT;
    const char* at[N]; const char* mk[MASK ? N : 1];
    u32x4 v[N], y[MASK ? N : 1];
    __device__ __forceinline__ void load(int q0, int q_end) {
        const int q = q0 + (threadIdx.x & 7) * 8;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool ok = at[i] && q < q_end;
            v[i] = ok ? *reinterpret_cast<const u32x4*>(at[i] + (int64_t)q * 2) : u32x4{0, 0, 0, 0};
            if (MASK) y[i] = ok ? *reinterpret_cast<const u32x4*>(mk[i] + (int64_t)q * 2) : u32x4{0, 0, 0, 0};
        }
    }
    __device__ __forceinline__ void store(char* lds) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (MASK)
#pragma unroll
                for (int w = 0; w < 4; ++w) v[i][w] = keep_where(v[i][w], y[i][w]);
            const int id = threadIdx.x + i * NT;
            *reinterpret_cast<u32x4*>(lds + lds_piece(id >> 3, id & 7)) = v[i];
        }
    }
};

template <int ROWS, int NT, bool MASK>
struct AcrossQ {                     // the other index contiguous in memory
    static constexpr int ITEMS = ROWS * 2, N = (ITEMS + NT - 1) / NT;
    u32x4 v[N][4], y[MASK ? N : 1][4];
    // at(q) -> address of the row of q (NULL: nothing there); m: first index of the tile, m_end: its extent
    template <class At, class Mk>
    __device__ __forceinline__ void load(int q0, int q_end, int m, int m_end, At at, Mk mk) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = threadIdx.x + i * NT, m8 = id % (ROWS / 8), q4 = id / (ROWS / 8);
            const bool in = (ITEMS % NT == 0 || id < ITEMS) && m + m8 * 8 < m_end;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int q = q0 + q4 * 4 + r;
                const char* src = in && q < q_end ? at(q) : nullptr;
                v[i][r] = src ? *reinterpret_cast<const u32x4*>(src + (int64_t)(m + m8 * 8) * 2) : u32x4{0, 0, 0, 0};
                if (MASK) y[i][r] = src ? *reinterpret_cast<const u32x4*>(mk(q) + (int64_t)(m + m8 * 8) * 2) : u32x4{0, 0, 0, 0};
            }
        }
    }
    __device__ __forceinline__ void store(char* lds) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = threadIdx.x + i * NT, m8 = id % (ROWS / 8), q4 = id / (ROWS / 8);
            if (ITEMS % NT != 0 && id >= ITEMS) continue;
            if (MASK)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int w = 0; w < 4; ++w) v[i][r][w] = keep_where(v[i][r][w], y[i][r][w]);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t sel = h ? 0x07060302u : 0x05040100u;
                    const u32x2 o = {__builtin_amdgcn_perm(v[i][1][w], v[i][0][w], sel), __builtin_amdgcn_perm(v[i][3][w], v[i][2][w], sel)};
                    *reinterpret_cast<u32x2*>(lds + lds_piece(m8 * 8 + w * 2 + h, q4 >> 1) + (q4 & 1) * 8) = o;
                }
            }
        }
    }
};

// (expert, first row, end) of row tile `tile`; expert E: the rows behind the last segment; false: there is no such tile
__device__ __forceinline__ bool find_tile(const int32_t* __restrict__ offsets, int E, int R, int rows, int tile, int& e, int& a, int& b) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int e0 = 0; e0 <= E; e0 += kWave) {
        int sa = 0, sb = 0;
        if (e0 + lane < E) segment(offsets, e0 + lane, R, sa, sb);
        else if (e0 + lane == E) { sa = min(max(offsets[E], 0), R); sb = R; }
        const int n = (sb - sa + rows - 1) / rows;
        int incl = n;
        for (int o = 1; o < kWave; o <<= 1) { const int v = __shfl_up(incl, o); if (lane >= o) incl += v; }
        const int total = __builtin_amdgcn_readlane(incl, 63);
        if (tile < base + total) {
            const int l = __ffsll((unsigned long long)__ballot(base + incl > tile)) - 1;
            e = e0 + l;
            a = __builtin_amdgcn_readlane(sa, l) + (tile - base - (__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(n, l))) * rows;
            b = min(a + rows, __builtin_amdgcn_readlane(sb, l));
            return true;
        }
        base += total;
    }
    return false;
}

template <typename T, int MODE, int TM, int TC, int WM, int WC, bool MASK, bool F32>
__global__ __launch_bounds__(WM * WC * kWave) void expert_linear_kernel(LinArgs g) {
    constexpr int NT = WM * WC * kWave, FM = TM / WM / 16, FC = TC / WC / 16, STAGE = (TM + TC) * 128;
    extern __shared__ __attribute__((aligned(16))) char lin_lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave % WM, wc = wave / WM;
    int e, a, b, m0, c0 = 0, split = 0;
    if (MODE == LIN_DW) {
        int id = blockIdx.x;
        m0 = (id % g.m_tiles) * TM; id /= g.m_tiles;
        c0 = (id % g.c_tiles) * TC; id /= g.c_tiles;
        e = id % g.E; split = id / g.E;
        segment(g.offsets, e, g.R, a, b);
        if (g.splits > 1) {
            const int len = ((b - a + g.splits - 1) / g.splits + LIN_BQ - 1) / LIN_BQ * LIN_BQ;
            a = (int)min((int64_t)a + (int64_t)split * len, (int64_t)b);
            b = min(a + len, b);
        }
    } else {
        m0 = (blockIdx.x % g.m_tiles) * TM;
        if (!find_tile(g.offsets, g.E, g.R, TC, blockIdx.x / g.m_tiles, e, a, b)) return;
    }
    const bool nothing = MODE != LIN_DW && e == g.E;
    const T* P = reinterpret_cast<const T*>(g.p) + (MODE != LIN_DW && !nothing ? e * g.p_expert : 0);
    const T* Q = reinterpret_cast<const T*>(g.q);
    const T* Y = reinterpret_cast<const T*>(g.mask);
    const int q_begin = MODE == LIN_DW ? a : 0, q_end = MODE == LIN_DW ? b : (nothing ? 0 : g.K);

    f32x4 acc[FM][FC];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FC; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    typedef typename std::conditional<MODE == LIN_FWD, AlongQ<TM, NT, false>, AcrossQ<TM, NT, false>>::type StageP;
    typedef typename std::conditional<MODE == LIN_DW, AcrossQ<TC, NT, MASK>, AlongQ<TC, NT, MASK>>::type StageQ;
    StageP sp;
    StageQ sq;
    if constexpr (MODE == LIN_FWD) {
#pragma unroll
        for (int i = 0; i < StageP::N; ++i) {
            const int m = m0 + ((threadIdx.x + i * NT) >> 3);
            sp.at[i] = m < g.M ? reinterpret_cast<const char*>(P + (int64_t)m * g.ldp) : nullptr;
        }
    }
    if constexpr (MODE != LIN_DW) {
#pragma unroll
        for (int i = 0; i < StageQ::N; ++i) {
            const int p = a + ((threadIdx.x + i * NT) >> 3);
            const char *src = nullptr, *my = nullptr;
            if (p < b && !nothing) {
                int row = p;
                if (MODE == LIN_FWD && g.rows) { row = g.rows[p]; row = row >= 0 ? g.top_k(row) : g.x_rows; }
                if (MODE != LIN_FWD || (unsigned)row < (unsigned)g.x_rows) src = reinterpret_cast<const char*>(Q + (int64_t)row * g.ldq);
                if (MASK) my = reinterpret_cast<const char*>(Y + (int64_t)row * g.ldmask);
            }
            sq.at[i] = src;
            if (MASK) sq.mk[i] = my;
        }
    }
    auto load = [&](int q0) {
        if constexpr (MODE == LIN_FWD) sp.load(q0, q_end);
        else if constexpr (MODE == LIN_DX)
            sp.load(q0, q_end, m0, g.M, [&](int q) { return reinterpret_cast<const char*>(P + (int64_t)q * g.ldp); }, [](int) { return (const char*)nullptr; });
        else
            sp.load(q0, q_end, m0, g.M, [&](int q) {
                int row = q;
                if (g.rows) { row = g.rows[q]; row = row >= 0 ? g.top_k(row) : g.x_rows; }
                return (unsigned)row < (unsigned)g.x_rows ? reinterpret_cast<const char*>(P + (int64_t)row * g.ldp) : nullptr;
            }, [](int) { return (const char*)nullptr; });
        if constexpr (MODE == LIN_DW)
            sq.load(q0, q_end, c0, g.C, [&](int q) { return reinterpret_cast<const char*>(Q + (int64_t)q * g.ldq); },
                    [&](int q) { return reinterpret_cast<const char*>(Y + (int64_t)q * g.ldmask); });
        else sq.load(q0, q_end);
    };
    auto store = [&](int buf) { sp.store(lin_lds + buf * STAGE); sq.store(lin_lds + buf * STAGE + TM * 128); };

    if (q_begin < q_end) {
        load(q_begin);
        store(0);
        __syncthreads();
        int buf = 0;
        for (int q0 = q_begin; q0 < q_end; q0 += LIN_BQ) {
            const bool more = q0 + LIN_BQ < q_end;
            if (more) load(q0 + LIN_BQ);
            const char* lp = lin_lds + buf * STAGE;
            const char* lq = lp + TM * 128;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                u32x4 fp[FM], fq[FC];
#pragma unroll
                for (int i = 0; i < FM; ++i)
                    fp[i] = *reinterpret_cast<const u32x4*>(lp + lds_piece(wm * (TM / WM) + i * 16 + (lane & 15), s * 4 + (lane >> 4)));
#pragma unroll
                for (int j = 0; j < FC; ++j)
                    fq[j] = *reinterpret_cast<const u32x4*>(lq + lds_piece(wc * (TC / WC) + j * 16 + (lane & 15), s * 4 + (lane >> 4)));
#pragma unroll
                for (int i = 0; i < FM; ++i)
#pragma unroll
                    for (int j = 0; j < FC; ++j) acc[i][j] = mfma16<T>(fp[i], fq[j], acc[i][j]);
            }
            if (more) store(buf ^ 1);
            __syncthreads();
            buf ^= 1;
        }
    }

    const int c_base = wc * (TC / WC) + (lane & 15), m_base = m0 + wm * (TM / WM) + (lane >> 4) * 4;
#pragma unroll
    for (int j = 0; j < FC; ++j) {
        const int c = MODE == LIN_DW ? c0 + c_base + j * 16 : a + c_base + j * 16;
        if (c >= (MODE == LIN_DW ? g.C : b)) continue;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
            const int m = m_base + i * 16;
            if (m >= g.M) continue;
            f32x4 v = acc[i][j];
            if (MODE == LIN_FWD && g.relu)
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = v[r] <= 0.f ? 0.f : v[r];         // (NaN stays)
            if (MODE == LIN_DW && g.splits > 1) {
                *reinterpret_cast<f32x4*>(g.partial + (((int64_t)split * g.E + e) * g.C + c) * g.M + m) = v;
            } else if (F32) {
                *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(g.d) + e * g.d_expert + (int64_t)c * g.ldd + m) = v;
            } else {
                typename Elem<T>::x4 o;
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = (T)v[r];
                *reinterpret_cast<typename Elem<T>::x4*>(reinterpret_cast<T*>(g.d) + (MODE == LIN_DW ? e * g.d_expert : 0) + (int64_t)c * g.ldd + m) = o;
            }
        }
    }
}

// sums of the splits, in the order of the splits
template <typename T>
__global__ __launch_bounds__(256) void expert_sum_splits_kernel(const float* __restrict__ part, int splits, int64_t n, T* __restrict__ d) {
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
        f32x4 s = *reinterpret_cast<const f32x4*>(part + i);
        for (int q = 1; q < splits; ++q) s += *reinterpret_cast<const f32x4*>(part + q * n + i);
#pragma unroll
        for (int r = 0; r < 4; ++r) d[i + r] = (T)s[r];
    }
}

static int lin_check(const char* what, int dtype, int n_in, int n_out, int E, int64_t R, int top_k, const int32_t* offsets) {
    NSX_REQUIRE(dtype == NSX_DTYPE_F16 || dtype == NSX_DTYPE_BF16, "%s: dtype %d is not a 16-bit float", what, dtype);
    NSX_REQUIRE(E >= 1 && E <= NSX_MAX_EXPERTS, "%s: n_experts %d not in [1,%d]", what, E, NSX_MAX_EXPERTS);
    NSX_REQUIRE(top_k >= 1 && top_k <= NSX_MAX_TOP_K, "%s: top_k %d not in [1,%d]", what, top_k, NSX_MAX_TOP_K);
    NSX_REQUIRE(R >= 0 && R <= NSX_MAX_EXPERT_ENTRIES, "%s: %lld ordered rows", what, (long long)R);
    NSX_REQUIRE(n_in >= 8 && n_in % 8 == 0 && n_in <= NSX_MAX_EXPERT_WIDTH && n_out >= 8 && n_out % 8 == 0 && n_out <= NSX_MAX_EXPERT_WIDTH,
                "%s: widths %d -> %d are not multiples of 8 in [8,%d]", what, n_in, n_out, NSX_MAX_EXPERT_WIDTH);
    NSX_REQUIRE(offsets, "%s: NULL offsets", what);
    return NSX_OK;
}

template <typename T, int MODE, int TM, int TC, int WM, int WC, bool F32>
static void lin_launch(const LinArgs& g, int64_t blocks, hipStream_t st) {
    constexpr int lds = 2 * (TM + TC) * 128;
    if (g.mask) expert_linear_kernel<T, MODE, TM, TC, WM, WC, true, F32><<<(unsigned)blocks, WM * WC * kWave, lds, st>>>(g);
    else expert_linear_kernel<T, MODE, TM, TC, WM, WC, false, F32><<<(unsigned)blocks, WM * WC * kWave, lds, st>>>(g);
}

static int64_t row_tiles(int64_t R, int E, int rows) { return R / rows + E + 1; }

static int dw_splits(int64_t R, int E, int n_in, int n_out) {
    const int64_t tiles = (int64_t)E * ((n_in + 63) / 64) * ((n_out + 63) / 64);
    int64_t s = (4 * (int64_t)num_cus() + tiles - 1) / tiles;
    const int64_t most = R / ((int64_t)E * 256);
    if (s > most) s = most;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

}  // namespace nsx

extern "C" {

int nsx_expert_linear_fwd(const void* x, int dtype, int64_t x_stride, int64_t x_rows, const int32_t* rows, int top_k,
                          const void* weight, int n_in, int n_out, int E, const int32_t* offsets, int64_t R, int relu, void* y,
                          void* stream) {
    using namespace nsx;
    const int rc = lin_check("nsx_expert_linear_fwd", dtype, n_in, n_out, E, R, top_k, offsets);
    if (rc != NSX_OK) return rc;
    if (R == 0) return NSX_OK;
    NSX_REQUIRE(weight && y && (x || x_rows == 0) && aligned16(x) && aligned16(weight) && aligned16(y) && x_stride >= n_in && x_stride % 8 == 0,
                "nsx_expert_linear_fwd: NULL or unaligned pointer or row stride %lld", (long long)x_stride);
    NSX_REQUIRE(x_rows >= 0 && x_rows <= NSX_MAX_EXPERT_ENTRIES && (rows || x_rows == R), "nsx_expert_linear_fwd: x has %lld rows", (long long)x_rows);
    LinArgs g{};
    g.p = weight; g.q = x; g.d = y; g.ldp = n_in; g.ldq = x_stride; g.ldd = n_out; g.p_expert = (int64_t)n_in * n_out;
    g.offsets = offsets; g.rows = rows; g.top_k = fast_div(top_k); g.E = E; g.R = (int)R; g.x_rows = (int)x_rows;
    g.M = n_out; g.K = n_in; g.relu = relu; g.m_tiles = (n_out + 63) / 64;
    const int64_t blocks = row_tiles(R, E, 64) * g.m_tiles;
    NSX_REQUIRE(blocks <= 0x7fffffff, "nsx_expert_linear_fwd: %lld tiles", (long long)blocks);
    if (dtype == NSX_DTYPE_F16) lin_launch<half_t, LIN_FWD, 64, 64, 2, 2, false>(g, blocks, (hipStream_t)stream);
    else lin_launch<bf16_t, LIN_FWD, 64, 64, 2, 2, false>(g, blocks, (hipStream_t)stream);
    NSX_LAUNCH_CHECK("nsx_expert_linear_fwd");
    return NSX_OK;
}

int nsx_expert_linear_bwd_x(const void* dy, int dtype, int64_t dy_stride, const void* y, int64_t y_stride, const void* weight,
                            int n_in, int n_out, int E, const int32_t* offsets, int64_t R, void* dx, void* stream) {
    using namespace nsx;
    const int rc = lin_check("nsx_expert_linear_bwd_x", dtype, n_in, n_out, E, R, 1, offsets);
    if (rc != NSX_OK) return rc;
    if (R == 0) return NSX_OK;
    NSX_REQUIRE(dy && weight && dx && aligned16(dy) && aligned16(y) && aligned16(weight) && aligned16(dx) && dy_stride >= n_out &&
                    dy_stride % 8 == 0 && (!y || (y_stride >= n_out && y_stride % 8 == 0)),
                "nsx_expert_linear_bwd_x: NULL or unaligned pointer or row stride");
    LinArgs g{};
    g.p = weight; g.q = dy; g.mask = y; g.d = dx; g.ldp = n_in; g.ldq = dy_stride; g.ldmask = y_stride; g.ldd = n_in;
    g.p_expert = (int64_t)n_in * n_out; g.offsets = offsets; g.E = E; g.R = (int)R; g.x_rows = (int)R;
    g.M = n_in; g.K = n_out; g.m_tiles = (n_in + 63) / 64;
    const int64_t blocks = row_tiles(R, E, 64) * g.m_tiles;
    NSX_REQUIRE(blocks <= 0x7fffffff, "nsx_expert_linear_bwd_x: %lld tiles", (long long)blocks);
    if (dtype == NSX_DTYPE_F16) lin_launch<half_t, LIN_DX, 64, 64, 2, 2, false>(g, blocks, (hipStream_t)stream);
    else lin_launch<bf16_t, LIN_DX, 64, 64, 2, 2, false>(g, blocks, (hipStream_t)stream);
    NSX_LAUNCH_CHECK("nsx_expert_linear_bwd_x");
    return NSX_OK;
}

int64_t nsx_expert_linear_bwd_w_workspace(int64_t R, int E, int n_in, int n_out) {
    using namespace nsx;
    int32_t some = 0;
    const int rc = lin_check("nsx_expert_linear_bwd_w_workspace", NSX_DTYPE_F16, n_in, n_out, E, R, 1, &some);
    if (rc != NSX_OK) return rc;
    const int s = dw_splits(R, E, n_in, n_out);
    return s > 1 ? (int64_t)s * E * n_in * n_out * 4 : 0;
}

int nsx_expert_linear_bwd_w(const void* x, int dtype, int64_t x_stride, int64_t x_rows, const int32_t* rows, int top_k,
                            const void* dy, int64_t dy_stride, const void* y, int64_t y_stride, int n_in, int n_out, int E,
                            const int32_t* offsets, int64_t R, int dw_f32, void* dw, void* workspace, void* stream) {
    using namespace nsx;
    const int rc = lin_check("nsx_expert_linear_bwd_w", dtype, n_in, n_out, E, R, top_k, offsets);
    if (rc != NSX_OK) return rc;
    NSX_REQUIRE(dw && aligned16(dw) && (R == 0 || dy) && (x || x_rows == 0) && aligned16(x) && aligned16(dy) && aligned16(y) && x_stride >= n_in &&
                    x_stride % 8 == 0 && dy_stride >= n_out && dy_stride % 8 == 0 && (!y || (y_stride >= n_out && y_stride % 8 == 0)),
                "nsx_expert_linear_bwd_w: NULL or unaligned pointer or row stride");
    NSX_REQUIRE(x_rows >= 0 && x_rows <= NSX_MAX_EXPERT_ENTRIES && (rows || x_rows == R), "nsx_expert_linear_bwd_w: x has %lld rows", (long long)x_rows);
    LinArgs g{};
    g.splits = dw_splits(R, E, n_in, n_out);
    NSX_REQUIRE(g.splits == 1 || (workspace && aligned16(workspace)), "nsx_expert_linear_bwd_w: no workspace");
    g.p = x; g.q = dy; g.mask = y; g.d = dw; g.ldp = x_stride; g.ldq = dy_stride; g.ldmask = y_stride; g.ldd = n_in;
    g.d_expert = (int64_t)n_in * n_out; g.offsets = offsets; g.rows = rows; g.top_k = fast_div(top_k); g.E = E; g.R = (int)R;
    g.x_rows = (int)x_rows; g.M = n_in; g.C = n_out; g.m_tiles = (n_in + 63) / 64; g.c_tiles = (n_out + 63) / 64;
    g.partial = (float*)workspace;
    const int64_t blocks = (int64_t)E * g.m_tiles * g.c_tiles * g.splits, n = (int64_t)E * n_in * n_out;
    NSX_REQUIRE(blocks <= 0x7fffffff, "nsx_expert_linear_bwd_w: %lld tiles", (long long)blocks);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == NSX_DTYPE_F16) {
        if (dw_f32) lin_launch<half_t, LIN_DW, 64, 64, 2, 2, true>(g, blocks, st);
        else lin_launch<half_t, LIN_DW, 64, 64, 2, 2, false>(g, blocks, st);
    } else {
        if (dw_f32) lin_launch<bf16_t, LIN_DW, 64, 64, 2, 2, true>(g, blocks, st);
        else lin_launch<bf16_t, LIN_DW, 64, 64, 2, 2, false>(g, blocks, st);
    }
    NSX_LAUNCH_CHECK("nsx_expert_linear_bwd_w");
    if (g.splits > 1) {
        const int64_t need = (n / 4 + 255) / 256, most = (int64_t)num_cus() * 8;
        const unsigned grid = (unsigned)(need < most ? need : most);
        if (dw_f32) expert_sum_splits_kernel<float><<<grid, 256, 0, st>>>(g.partial, g.splits, n, (float*)dw);
        else if (dtype == NSX_DTYPE_F16) expert_sum_splits_kernel<half_t><<<grid, 256, 0, st>>>(g.partial, g.splits, n, (half_t*)dw);
        else expert_sum_splits_kernel<bf16_t><<<grid, 256, 0, st>>>(g.partial, g.splits, n, (bf16_t*)dw);
        NSX_LAUNCH_CHECK("nsx_expert_linear_bwd_w");
    }
    return NSX_OK;
}

}  // extern "C"
