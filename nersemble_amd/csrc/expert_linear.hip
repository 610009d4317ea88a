// expert_linear.hip -- routed experts: every ordered row times the weight matrix of its expert, and the two gradients.
//
//   y_p = act(W_e x_r(p)),   dx_p = W_e^T dz_p,   dW_e = sum_{p in e} dz_p x_r(p)^T,   dz = dy where y > 0 (ReLU) or dy
//
// All three are D[m][c] = sum_q P[m][q] Q[c][q] with m the index that is contiguous in memory in the result:
//   forward  m = output feature, c = ordered row,      q = input feature    P = W (q contiguous)  Q = x (q contiguous)
//   dx       m = input feature,  c = ordered row,      q = output feature   P = W (m contiguous)  Q = dz (q contiguous)
//   dW       m = input feature,  c = output feature,   q = ordered row      P = x (m contiguous)  Q = dz (c contiguous)
// One kernel: a workgroup makes a TM x TC tile in steps of 64 q.  16-bit tiles of P and Q lie in LDS with q contiguous;
// v_mfma_f32_32x32x16 with 32-bit accumulators, a wave's tile up to 128 x 64.  What is not q-contiguous in memory is turned on
// its way through the registers: 4 q x 8 m per thread, 16 byte permutations, eight 8-byte stores.
//   * One LDS buffer and two or three workgroups per CU: while one stores its next tile and waits, another multiplies.  (Two
//     buffers with one barrier per step, one workgroup of 8 waves and a 256 x 256 tile came to the same rate within 5 %, at a
//     coarser grain: ragged segments and the last round of workgroups cost more.)
//   * A step's global loads are issued under the first quarter of the previous step's products and stay in flight through
//     them.  The fragments of a quarter step are read while its predecessor is multiplied, a P fragment into the registers of
//     the one just used: 32 x 32 x 16 products need half the fragment registers of 16 x 16 x 32 (which spilled).
//   * 16-bit results leave through LDS as whole rows.
// Segments are read from the plan on the device: the grid covers the most tiles that any split of R rows over E experts can
// have, every workgroup finds its (expert, tile) by one scan of the offsets.
#include "expert_common.h"
#include <algorithm>
#include <type_traits>

namespace nsx {

typedef float f32x16 __attribute__((ext_vector_type(16)));
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
    int m_tiles, c_tiles, relu;
    int chunk;                       // dW: rows per partial sum (0: a whole segment, no partial sums)
    float* partial;                  // [chunk][C][M]
    const void* x; int64_t ldx;      // narrow layers: both gradients at once
};

template <typename T> __device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mfma32<half_t>(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(Elem<half_t>::x8, a), __builtin_bit_cast(Elem<half_t>::x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma32<bf16_t>(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Elem<bf16_t>::x8, a), __builtin_bit_cast(Elem<bf16_t>::x8, b), c, 0, 0, 0);
}

constexpr int LIN_BQ = 64;           // q per step: rows of 128 B in LDS
constexpr uint32_t lin_rows(uint32_t rows) { return rows * 128; }
// Byte of a 16-byte piece of a row.  The permutation: a phase of a fragment read takes 16 rows (half of the 64 banks each), and
// the turned stores take rows 8 apart -- both have to fall on different banks.
__device__ __forceinline__ uint32_t lin_piece(int row, int ch) { return row * 128 + ((ch ^ (row >> 1) ^ ((row >> 4) & 3)) & 7) * 16; }

// both 16-bit halves of `v` kept where those of `y` (not negative) are not zero
__device__ __forceinline__ uint32_t keep_where(uint32_t v, uint32_t y) {
    const uint32_t t = ((y & 0x7fff7fffu) + 0x7fff7fffu) & 0x80008000u;
    return v & (t | (t - (t >> 15)));
}

// 0 for gathered rows that are not there: what is loaded without a branch is loaded from here
__device__ u32x4 lin_zeros;
__device__ __forceinline__ const char* zero_row() { return reinterpret_cast<const char*>(&lin_zeros); }
__device__ __forceinline__ u32x4 load16(const char* p) { return *reinterpret_cast<const u32x4*>(p); }
// reads behind `bytes` give 0
__device__ __forceinline__ __amdgpu_buffer_rsrc_t lin_buffer(const char* p, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(p), 0, (int)min(bytes, (int64_t)0x7fffffff), 0x00020000);
}
__device__ __forceinline__ u32x4 lin_load(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0));
}

// ---- which tile ---------------------------------------------------------------------------------------------------
// row tiles of all segments and of the rows behind the last one
__device__ __forceinline__ int count_tiles(const int32_t* __restrict__ offsets, int E, int R, int rows) {
    int n = 0;
    for (int e = threadIdx.x & 63; e <= E; e += kWave) {
        int a, b;
        if (e < E) segment(offsets, e, R, a, b);
        else { a = min(max(offsets[E], 0), R); b = R; }
        n += (b - a + rows - 1) / rows;
    }
    for (int o = 1; o < kWave; o <<= 1) n += __shfl_xor(n, o);
    return __builtin_amdgcn_readfirstlane(n);
}
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
            const int start = __builtin_amdgcn_readlane(sa, l), end = __builtin_amdgcn_readlane(sb, l);
            a = start + (tile - base - (__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(n, l))) * rows;
            b = min(a + rows, end);
            return a >= start && a < b;                    // (always, of a plan's offsets)
        }
        base += total;
    }
    return false;
}
// Consecutive workgroups go to the 8 XCDs in turn; those that run on one at a time should share what they read through its L2.
// Forward and dx: each XCD takes a stretch of its own of an order in which 8 row tiles pass through all m tiles.
constexpr int LIN_GROUP = 8;
__device__ __forceinline__ bool lin_order(int tiles, int m_tiles, int block, int& tile, int& m) {
    const int64_t all = (int64_t)tiles * m_tiles, per = (all + 7) / 8, id = (block & 7) * per + (block >> 3);
    if ((block >> 3) >= per || id >= all) return false;
    const int group = (int)(id / (LIN_GROUP * m_tiles)), rest = (int)(id - (int64_t)group * (LIN_GROUP * m_tiles));
    const int n = min(LIN_GROUP, tiles - group * LIN_GROUP);
    m = rest / n;
    tile = group * LIN_GROUP + rest - m * n;
    return true;
}
// The expert with the rank-th most rows (up to 64 experts; of more, simply the rank-th): the longest sums start first and do not
// end alone.
__device__ __forceinline__ int expert_by_size(const int32_t* __restrict__ offsets, int E, int R, int rank) {
    if (E > kWave) return rank;
    const int lane = threadIdx.x & 63;
    int a = 0, b = 0;
    if (lane < E) segment(offsets, lane, R, a, b);
    const int n = b - a;
    int before = 0;
    for (int e = 0; e < E; ++e) {
        const int other = __builtin_amdgcn_readlane(n, e);
        before += (other > n || (other == n && e < lane)) ? 1 : 0;
    }
    return __ffsll((unsigned long long)__ballot(lane < E && before == rank)) - 1;
}
// dW: an XCD takes blocks of up to 4 x 4 tiles of one segment (or chunk of one) in turn with the others.  (No workgroups for
// tiles that are not there: of blocks of 16 with one tile each, the working ones fell on two of an XCD's 32 CUs.)
__host__ __device__ __forceinline__ int lin_group_dw(int tiles) { return tiles < 4 ? tiles : 4; }
__device__ __forceinline__ bool lin_order_dw(const LinArgs& g, int block, int& s, int& m, int& c) {
    const int wm = lin_group_dw(g.m_tiles), wc = lin_group_dw(g.c_tiles), gm = (g.m_tiles + wm - 1) / wm, gc = (g.c_tiles + wc - 1) / wc;
    const int local = block >> 3, within = local % (wm * wc);
    int group = local / (wm * wc) * 8 + (block & 7);
    m = group % gm * wm + within % wm; group /= gm;
    c = group % gc * wc + within / wm;
    s = group / gc;
    return m < g.m_tiles && c < g.c_tiles;
}

// ---- the products -------------------------------------------------------------------------------------------------
template <typename T, int MODE, int TM, int TC, int WM, int WC, bool MASK, bool F32>
__global__ __launch_bounds__(WM * WC * kWave, 2) void expert_linear_kernel(LinArgs g) {
    extern __shared__ __attribute__((aligned(16))) char lin_lds[];
    constexpr bool P_ALONG = MODE == LIN_FWD, Q_ALONG = MODE != LIN_DW;
    constexpr int NT = WM * WC * kWave, FM = TM / WM / 32, FC = TC / WC / 32, NP = TM * 8 / NT, NQ = TC * 8 / NT, RPT = NT / 8;
    constexpr uint32_t Q_AT = lin_rows(TM);
    static_assert(NT >= 128 && (P_ALONG || NP % 4 == 0) && (Q_ALONG || NQ % 4 == 0), "a thread turns 4 rows of q");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave % WM, wc = wave / WM;
    int e, a, b, m0, c0 = 0, chunk = 0;
    if (MODE == LIN_DW) {
        if (!lin_order_dw(g, blockIdx.x, chunk, m0, c0)) return;
        m0 *= TM; c0 *= TC;
        if (g.chunk > 0) {
            if (chunk >= g.R / g.chunk + g.E || !find_tile(g.offsets, g.E, g.R, g.chunk, chunk, e, a, b) || e == g.E) return;
        } else {
            if (chunk >= g.E) return;
            e = expert_by_size(g.offsets, g.E, g.R, chunk);
            segment(g.offsets, e, g.R, a, b);
        }
    } else {
        int tile;
        if (!lin_order(count_tiles(g.offsets, g.E, g.R, TC), g.m_tiles, blockIdx.x, tile, m0)) return;
        m0 *= TM;
        if (!find_tile(g.offsets, g.E, g.R, TC, tile, e, a, b)) return;
    }
    const bool nothing = MODE != LIN_DW && e == g.E;
    const char* P = reinterpret_cast<const char*>(g.p) + (MODE != LIN_DW && !nothing ? e * g.p_expert * 2 : 0);
    const char* Q = reinterpret_cast<const char*>(g.q);
    const char* Y = reinterpret_cast<const char*>(g.mask);
    const int q_begin = MODE == LIN_DW ? a : 0, q_end = MODE == LIN_DW ? b : (nothing ? 0 : g.K);

    f32x16 acc[FM][FC];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FC; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

    // Global reads.  Along q: rows tid / 8 + RPT i, piece tid % 8; across q: pieces tid % (rows / 8) of rows of q, 4 to a thread.
    // What has no rows to gather goes through a buffer descriptor whose range ends where the data does (0 behind it).
    constexpr int PM = TM / 8, QC = TC / 8;
    const int pm = min(m0 + (tid % PM) * 8, g.M - 8) * 2, qc = min(c0 + (tid % QC) * 8, g.C - 8) * 2;
    const uint32_t q_row = (uint32_t)g.ldq * 2, y_row = (uint32_t)g.ldmask * 2, p_row = (uint32_t)g.ldp * 2;
    auto quad = [&](int rows8, int k) { return (tid / rows8 + k * (NT / rows8)) ^ (rows8 >= 16 ? (tid >> 3) & 1 : 0); };
    auto p_across = [&](int i) { return quad(PM, i >> 2) * 4 + (i & 3); };
    auto q_across = [&](int i) { return quad(QC, i >> 2) * 4 + (i & 3); };
    constexpr int NROW = MODE == LIN_FWD ? NQ : MODE == LIN_DW ? NP : 1;
    int row[NROW];                               // gathered rows: of Q (forward), of P one step ahead (dW)
    if (MODE == LIN_FWD)
#pragma unroll
        for (int i = 0; i < NROW; ++i) {
            const int p = min(a + (tid >> 3) + RPT * i, b - 1);
            row[i] = p;
            if (g.rows) { row[i] = g.rows[p]; row[i] = row[i] >= 0 ? g.top_k(row[i]) : -1; }
            if (row[i] >= g.x_rows) row[i] = -1;
        }
    auto locate = [&](int q0) {                  // (the entry as it is: what follows from it is computed where it is used)
        if (MODE == LIN_DW)
#pragma unroll
            for (int r = 0; r < NROW; ++r) {
                const int q = min(q0 + p_across(r), q_end - 1);
                row[r] = g.rows ? g.rows[q] : q;
            }
    };
    auto row_of = [&](int q, int r) {
        int v = row[r];
        if (g.rows) v = v >= 0 ? g.top_k(v) : -1;
        return q < q_end && v < g.x_rows ? v : -1;
    };
    u32x4 pv[NP], qv[NQ], yv[MASK ? NQ : 1];
    const auto p_buf = lin_buffer(P, MODE == LIN_DW ? 0 : (int64_t)g.p_expert * 2);
    const auto q_buf = lin_buffer(Q + (MODE == LIN_DX ? (int64_t)a * q_row : 0), MODE == LIN_DX ? (int64_t)(b - a) * q_row : 0);
    const auto y_buf = lin_buffer(MASK ? Y + (MODE == LIN_DX ? (int64_t)a * y_row : 0) : Q, MODE == LIN_DX ? (int64_t)(b - a) * y_row : 0);
    auto load_p = [&](int q0, int i) {
        const int q = q0 + (tid & 7) * 8;
        if (MODE == LIN_FWD) pv[i] = lin_load(p_buf, (uint32_t)(m0 + (tid >> 3) + RPT * i) * p_row + q * 2 | (q >= q_end ? 0x80000000u : 0u));
        else if (MODE == LIN_DX) pv[i] = lin_load(p_buf, (uint32_t)(q0 + p_across(i)) * p_row + pm);
        else {
            const int r = row_of(q0 + p_across(i), i);
            pv[i] = load16(r < 0 ? zero_row() : P + (uint64_t)(uint32_t)r * p_row + pm);
        }
    };
    auto load_q = [&](int q0, int i) {
        const int q = q0 + (tid & 7) * 8;
        const uint32_t past = q >= q_end ? 0x80000000u : 0u;         // (behind every range)
        if (MODE == LIN_FWD) qv[i] = load16(past || row[i] < 0 ? zero_row() : Q + (uint64_t)(uint32_t)row[i] * q_row + q * 2);
        else if (MODE == LIN_DX) {
            qv[i] = lin_load(q_buf, (uint32_t)((tid >> 3) + RPT * i) * q_row + q * 2 | past);
            if (MASK) yv[i] = lin_load(y_buf, (uint32_t)((tid >> 3) + RPT * i) * y_row + q * 2 | past);
        } else {
            const int64_t left = max(q_end - q0, 0);
            qv[i] = lin_load(lin_buffer(Q + (int64_t)q0 * q_row, left * q_row), (uint32_t)q_across(i) * q_row + qc);
            if (MASK) yv[i] = lin_load(lin_buffer(Y + (int64_t)q0 * y_row, left * y_row), (uint32_t)q_across(i) * y_row + qc);
        }
    };
    auto mask_q = [&](int i) {
        if (MASK)
#pragma unroll
            for (int w = 0; w < 4; ++w) qv[i][w] = keep_where(qv[i][w], yv[i][w]);
    };
    const uint32_t st_along = lin_piece(tid >> 3, tid & 7);
    auto put_across = [&](uint32_t base, int rows8, const u32x4* v, int i) {     // (v: 4 rows of q; i: which two of 8 rows of m or c)
        const int k = i >> 2, w = i & 3, q4 = quad(rows8, k);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t sel = h ? 0x07060302u : 0x05040100u;
            const u32x2 o = {__builtin_amdgcn_perm(v[k * 4 + 1][w], v[k * 4][w], sel), __builtin_amdgcn_perm(v[k * 4 + 3][w], v[k * 4 + 2][w], sel)};
            *reinterpret_cast<u32x2*>(lin_lds + base + lin_piece((tid % rows8) * 8 + w * 2 + h, q4 >> 1) + (q4 & 1) * 8) = o;
        }
    };
    auto put_p = [&](int i) {
        if (P_ALONG) *reinterpret_cast<u32x4*>(lin_lds + (st_along ^ (RPT * i >> 4 & 3) * 16) + i * lin_rows(RPT)) = pv[i];
        else put_across(0, PM, pv, i);
    };
    auto put_q = [&](int i) {
        if (Q_ALONG) *reinterpret_cast<u32x4*>(lin_lds + Q_AT + (st_along ^ (RPT * i >> 4 & 3) * 16) + i * lin_rows(RPT)) = qv[i];
        else put_across(Q_AT, QC, qv, i);
    };
    // fragments: row 32 i + (lane & 31) of the wave's rows, piece 2 s + lane / 32
    const uint32_t fr_p = wm * lin_rows(TM / WM), fr_q = Q_AT + wc * lin_rows(TC / WC);
    uint32_t fr[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) fr[s] = lin_piece(lane & 31, 2 * s + (lane >> 5));
    auto frag = [&](uint32_t at, int row0, int s, int i) {
        return *reinterpret_cast<const u32x4*>(lin_lds + at + (fr[s] ^ ((row0 >> 5) + i & 1) * 32) + i * lin_rows(32));
    };
    u32x4 fp[FM], fq[2][FC];

    // Which of a SIMD's waves goes first: the one that multiplies, so that one workgroup's stores fall under another's products; for
    // dx's large tiles (turning W takes longer) always the same one of two (its slot).  us without | so: 16384 x 2 of 16, 1024 -> 2048
    // forward 183 | 174, dW 180 | 169, dx 170 | 163;  8192 x 2, 1024 -> 1024  forward 57 | 53, dW 62 | 57;  masked dx 288 | 302: without
    constexpr int PRIO = MODE == LIN_DX && TM == 256 ? 2 : MODE == LIN_DX && MASK ? 0 : 1;
    if (PRIO == 2 && (__builtin_amdgcn_s_getreg(4 | 3 << 11) & 1)) __builtin_amdgcn_s_setprio(3);      // HW_ID, bits 3:0: the slot
    if (q_begin < q_end) {
        locate(q_begin);
#pragma unroll
        for (int i = 0; i < NP; ++i) load_p(q_begin, i);
#pragma unroll
        for (int i = 0; i < NQ; ++i) load_q(q_begin, i);
        locate(q_begin + LIN_BQ);
        for (int q0 = q_begin; q0 < q_end; q0 += LIN_BQ) {
            if (PRIO == 1) __builtin_amdgcn_s_setprio(0);
            if (q0 > q_begin) __syncthreads();
#pragma unroll
            for (int i = 0; i < NP; ++i) put_p(i);
#pragma unroll
            for (int i = 0; i < NQ; ++i) mask_q(i);
#pragma unroll
            for (int i = 0; i < NQ; ++i) put_q(i);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < FM; ++i) fp[i] = frag(fr_p, wm * (TM / WM), 0, i);
#pragma unroll
            for (int j = 0; j < FC; ++j) fq[0][j] = frag(fr_q, wc * (TC / WC), 0, j);
            if (PRIO == 1) __builtin_amdgcn_s_setprio(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int i = 0; i < FM; ++i) {
#pragma unroll
                    for (int j = 0; j < FC; ++j) acc[i][j] = mfma32<T>(fp[i], fq[s & 1][j], acc[i][j]);
                    if (s < 3) {
                        fp[i] = frag(fr_p, wm * (TM / WM), s + 1, i);
#pragma unroll
                        for (int j = i * FC / FM; j < (i + 1) * FC / FM; ++j) fq[(s + 1) & 1][j] = frag(fr_q, wc * (TC / WC), s + 1, j);
                    }
                    if (s == 0) {
#pragma unroll
                        for (int k = i * NP / FM; k < (i + 1) * NP / FM; ++k) load_p(q0 + LIN_BQ, k);
#pragma unroll
                        for (int k = i * NQ / FM; k < (i + 1) * NQ / FM; ++k) load_q(q0 + LIN_BQ, k);
                        if (i == FM - 1) locate(q0 + 2 * LIN_BQ);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
        }
    }

    const int c_first = (MODE == LIN_DW ? c0 : a) + wc * (TC / WC), c_end = MODE == LIN_DW ? g.C : b, m_first = m0 + wm * (TM / WM);
    if (F32) {
        float* D = MODE == LIN_DW && g.chunk > 0 ? g.partial + (int64_t)chunk * g.C * g.M : reinterpret_cast<float*>(g.d) + (MODE == LIN_DW ? e * g.d_expert : 0);
        const int64_t ldd = MODE == LIN_DW && g.chunk > 0 ? g.M : g.ldd;
#pragma unroll
        for (int j = 0; j < FC; ++j) {
            const int c = c_first + j * 32 + (lane & 31);
            if (c >= c_end) continue;
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int m = m_first + i * 32 + u * 8 + (lane >> 5) * 4;
                    if (m < g.M) *reinterpret_cast<f32x4*>(D + (int64_t)c * ldd + m) = f32x4{acc[i][j][u * 4], acc[i][j][u * 4 + 1], acc[i][j][u * 4 + 2], acc[i][j][u * 4 + 3]};
                }
        }
        return;
    }
    // 16-bit results: 32 rows of the wave's tile at a time through LDS, so that whole rows leave (as the lanes hold them they are
    // 16 bytes of each of 32 rows per instruction: 40 % of all requests to L2 at 1024 -> 2048, 8 % of the time)
    constexpr int ROW = TM / WM * 2 + 16, LPR = TM / WM / 8;                 // bytes per row in LDS; lanes per row
    char* mine = lin_lds + wave * 32 * ROW;
    T* D = reinterpret_cast<T*>(g.d) + (MODE == LIN_DW ? e * g.d_expert : 0);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < FC; ++j) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                typename Elem<T>::x4 o;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = acc[i][j][u * 4 + r];
                    if (MODE == LIN_FWD && g.relu) v = v <= 0.f ? 0.f : v;            // (NaN stays)
                    o[r] = (T)v;
                }
                *reinterpret_cast<typename Elem<T>::x4*>(mine + (lane & 31) * ROW + (i * 32 + u * 8 + (lane >> 5) * 4) * 2) = o;
            }
        wave_lds_fence();
#pragma unroll
        for (int k = 0; k < 32 * LPR / kWave; ++k) {
            const int r = k * (kWave / LPR) + lane / LPR, c = c_first + j * 32 + r, m = m_first + lane % LPR * 8;
            if (c < c_end && m < g.M)
                *reinterpret_cast<u32x4*>(D + (int64_t)c * g.ldd + m) = *reinterpret_cast<const u32x4*>(mine + r * ROW + lane % LPR * 16);
        }
        wave_lds_fence();
    }
}

// dW of an expert = the sum of its chunks, in their order: 16 of them side by side and 16 x 4 values per workgroup, or (few
// chunks) 256 x 4 values.  Bound by its chain of loads: 3.6 us for 700 chunks of 32 x 64 (5.7 MB), 4.3 for 81 of 176 x 136 (7.8 MB).
template <typename T>
__global__ __launch_bounds__(256) void expert_sum_chunks_kernel(LinArgs g, T* __restrict__ d) {
    __shared__ f32x4 part[16][16];
    const int e = blockIdx.y, lane = threadIdx.x & 63;
    int first = 0, a, b;
    for (int q = lane; q < e; q += kWave) { segment(g.offsets, q, g.R, a, b); first += (b - a + g.chunk - 1) / g.chunk; }
    for (int o = 1; o < kWave; o <<= 1) first += __shfl_xor(first, o);
    segment(g.offsets, e, g.R, a, b);
    const int n = min((b - a + g.chunk - 1) / g.chunk, g.R / g.chunk + g.E - first), ways = n > 8 ? 16 : 1;
    const int who = ways > 1 ? threadIdx.x >> 4 : 0, at = ways > 1 ? threadIdx.x & 15 : threadIdx.x, step = 1024 / ways;
    const int64_t size = (int64_t)g.C * g.M;
    for (int64_t i0 = (int64_t)blockIdx.x * step; i0 < size; i0 += (int64_t)gridDim.x * step) {
        const int64_t i = i0 + at * 4;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        if (i < size)
            for (int q = who; q < n; q += ways) s += *reinterpret_cast<const f32x4*>(g.partial + (first + q) * size + i);
        if (ways > 1) {
            part[who][at] = s;
            __syncthreads();
            if (who == 0)
                for (int q = 1; q < 16; ++q) s += part[q][at];
            __syncthreads();
        }
        if (who == 0 && i < size)
#pragma unroll
            for (int r = 0; r < 4; ++r) d[(int64_t)e * size + i + r] = (T)s[r];
    }
}

// ---- narrow layers: at most 64 m and 64 q ------------------------------------------------------------------------------
// Bound by memory: 32 -> 64 over 2^19 ordered rows reads 17 MB (from the caches, gathered) and writes 67.  No LDS and no barrier:
// a wave keeps the whole matrix of its expert as fragments, reads 64 rows straight into the other operand's and stores whole
// rows.  v_mfma_f32_16x16x32, D[m][c]: lane = row c of 16, four consecutive m per tile; the rows of P are dealt to the tiles so
// that a lane's 4 MT values are consecutive (m = (lane / 16) 4 MT + 4 t + r).
// us, tiles of 64 x 64 through LDS | this, 262144 rows x 2 of 16 experts, bf16 (dx with the ReLU's mask):
//   forward  32 -> 64  30.2 | 23.7   64 -> 64  30.1 | 29.1   64 -> 16  26.1 | 16.0   (100000 x 2 of 61: 128 -> 64  18.6 | 24.2)
//   dx       32 -> 64  35.9 | 27.7   64 -> 64  39.1 | 43.1   64 -> 16  28.7 | 22.8   16 -> 64  32.7 | 24.8   (in 16 bits)
// (dx gathers its matrix's fragments 2 bytes at a time, and with the mask's they leave fewer waves: up to 2048 weights.)
constexpr int NARROW_ROWS = 256;      // ordered rows per workgroup of 4 waves

template <typename T> __device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma16<half_t>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(Elem<half_t>::x8, a), __builtin_bit_cast(Elem<half_t>::x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<bf16_t>(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(Elem<bf16_t>::x8, a), __builtin_bit_cast(Elem<bf16_t>::x8, b), c, 0, 0, 0);
}

// An expert's matrix as fragments of P
template <typename T, int MODE, int MT, int QS>
__device__ __forceinline__ void narrow_matrix(const LinArgs& g, int e, u32x4 (&p)[MT][QS]) {
    const int lane = threadIdx.x & 63, c = lane & 15, piece = lane >> 4;
    const T* P = reinterpret_cast<const T*>(g.p) + e * g.p_expert;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = min((c >> 2) * (4 * MT) + t * 4 + (c & 3), g.M - 1);
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            const int at = s * 32 + piece * 8;
            if (MODE == LIN_FWD) p[t][s] = load16(at < g.K ? reinterpret_cast<const char*>(P + (int64_t)m * g.ldp + at) : zero_row());
            else {
                const uint16_t* w = reinterpret_cast<const uint16_t*>(P) + (int64_t)min(at, g.K - 8) * g.ldp + m;
                // (q behind the end: whatever is here meets zeros of the other operand -- unless it is not finite: cleared)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const uint32_t v = (uint32_t)w[(2 * h) * g.ldp] | (uint32_t)w[(2 * h + 1) * g.ldp] << 16;
                    p[t][s][h] = at < g.K ? v : 0u;
                }
            }
        }
    }
}
// 4 MT consecutive values of row `at`, from m on, in D (16 or 32 bits)
template <typename D, int MT>
__device__ __forceinline__ void narrow_store(const LinArgs& g, int at, const f32x4 (&acc)[MT], bool relu) {
    const int m = ((threadIdx.x & 63) >> 4) * (4 * MT);
    D* d = reinterpret_cast<D*>(g.d) + (int64_t)at * g.ldd + m;
    if constexpr (sizeof(D) == 4) {
#pragma unroll
        for (int t = 0; t < MT; ++t)
            if (m + t * 4 < g.M) *reinterpret_cast<f32x4*>(d + t * 4) = acc[t];
        return;
    }
    alignas(16) D out[4 * MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float v = acc[t][r];
            if (relu) v = v <= 0.f ? 0.f : v;                  // (NaN stays)
            out[t * 4 + r] = (D)v;
        }
    if (MT == 1) {
        if (m < g.M) *reinterpret_cast<u32x2*>(d) = *reinterpret_cast<const u32x2*>(out);
    } else
#pragma unroll
        for (int h = 0; h < MT / 2; ++h)
            if (m + h * 8 < g.M) *reinterpret_cast<u32x4*>(d + h * 8) = *reinterpret_cast<const u32x4*>(out + h * 8);
}

template <typename T, typename D, int MODE, int MT, int QS, bool MASK>
__global__ __launch_bounds__(4 * kWave) void expert_narrow_kernel(LinArgs g) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, piece = lane >> 4;
    int e, a, b;
    if (!find_tile(g.offsets, g.E, g.R, NARROW_ROWS, blockIdx.x, e, a, b)) return;
    a += wave * 64;
    if (a >= b) return;
    const bool nothing = e == g.E;
    // rows of this wave, one to a lane
    int row = min(a + lane, b - 1);
    if (MODE == LIN_FWD && g.rows) { row = g.rows[row]; row = row >= 0 ? g.top_k(row) : -1; }
    if (nothing || (MODE == LIN_FWD && row >= g.x_rows)) row = -1;
    const char* Q = reinterpret_cast<const char*>(g.q);
    const char* Y = reinterpret_cast<const char*>(g.mask);
    u32x4 q[4][QS], y[MASK ? 4 : 1][MASK ? QS : 1];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int r = __shfl(row, u * 16 + c);
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            const int at = s * 32 + piece * 8;
            const bool in = r >= 0 && at < g.K;
            q[u][s] = load16(in ? Q + ((int64_t)r * g.ldq + at) * 2 : zero_row());
            if (MASK) y[u][s] = load16(in ? Y + ((int64_t)r * g.ldmask + at) * 2 : zero_row());
        }
    }
    u32x4 p[MT][QS];
    narrow_matrix<T, MODE, MT, QS>(g, nothing ? 0 : e, p);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        if (a + u * 16 >= b) break;
        f32x4 acc[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < QS; ++s) {
            if (MASK)
#pragma unroll
                for (int w = 0; w < 4; ++w) q[u][s][w] = keep_where(q[u][s][w], y[u][s][w]);
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = mfma16<T>(p[t][s], q[u][s], acc[t]);
        }
        if (nothing)                                      // (the first expert's matrix may hold what is not finite)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (a + u * 16 + c < b) narrow_store<D, MT>(g, a + u * 16 + c, acc, MODE == LIN_FWD && g.relu);
    }
}

// Both gradients of a narrow layer in one pass over dy, y and x.  A wave takes 64 rows at a time: dz as fragments straight from
// memory, as in the kernel above, makes dx; for dW the rows are the sum's index, so dz and x go through LDS (a region of the wave's
// own) turned: a lane holds the same 8 features of the rows c, 16 + c, 32 + c and 48 + c, which it stores side by side -- the
// order of a sum over rows is free as long as both operands have it.  dW's 32-bit sums stay in registers for a whole chunk of a
// segment, the four waves' are added in their order at its end; expert_sum_chunks_kernel adds the chunks.
// Bound by memory: 262144 x 2 of 16 experts, 32 -> 64 with ReLU, dx in 32 bits: 52 us for 218 MB (4.2 TB/s); dx and dW apart read dy
// and y twice.  us, both gradients of gathered rows with the join and the sum of the chunks, apart | at once:
//   32 -> 64  89 | 66 (ReLU)  69 | 53 (none)    64 -> 64  142 | 124   109 | 110    64 -> 16  98 | 86    16 -> 64  73 | 48    64 -> 32  108 | 97
//   2048 rows x 2 of 16, 32 -> 64  18 | 12      100000 x 2 of 61, 32 -> 64  48 | 54, 64 -> 64  62 | 75 (chunks of two tiles: many are half full)
// Chunks for 2, 3, 4, 6 workgroups per CU, dx in 16 bits: 48.9, 46.3, 45.5, 47.9 (32 -> 64), without ReLU 30.8, 30.8, 29.9, 32.5.
// The widest tile's 64 KB of LDS and 240 to 270 registers leave room for one or two workgroups.  us, registers and chunks for three | for
// two, 64 -> 64 with ReLU: 262144 x 2 of 16  124 | 125;  2^20 x 2 of 4  458 | 483;  100000 x 2 of 61  75 | 69;  2^20 x 2 of 16, 48 -> 40
// 359 | 375: one rule for all tiles.
// Feature f's row of 128 bytes lies at f with the lowest bit turned by bit 3, its 16-byte pieces permuted by f / 2: neither the
// stores (features 8 apart) nor the fragment reads (16 features) meet on a bank.
__device__ __forceinline__ uint32_t turned_at(int f, int piece) { return (f ^ (f >> 3 & 1)) * 128 + ((piece ^ (f >> 1)) & 7) * 16; }
template <int S>
__device__ __forceinline__ void put_turned(char* lds, const u32x4 (&v)[4][S], int features) {
    const int lane = threadIdx.x & 63, c = lane & 15, piece = lane >> 4;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        if (s * 32 + piece * 8 >= features) continue;
#pragma unroll
        for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t sel = h ? 0x07060302u : 0x05040100u;
                const u32x2 o = {__builtin_amdgcn_perm(v[1][s][w], v[0][s][w], sel), __builtin_amdgcn_perm(v[3][s][w], v[2][s][w], sel)};
                *reinterpret_cast<u32x2*>(lds + turned_at(s * 32 + piece * 8 + w * 2 + h, c >> 1) + (c & 1) * 8) = o;
            }
    }
}

template <typename T, typename D, int MT, int QS, bool MASK>
__global__ __launch_bounds__(4 * kWave, 3) void expert_narrow_bwd_kernel(LinArgs g) {
    constexpr int XS = (MT + 1) / 2, CT = 2 * QS, MINE = (16 * MT + 32 * QS) * 128;
    static_assert(MT * CT * 1024 <= MINE, "the sums fit where the rows were");
    __shared__ __attribute__((aligned(16))) char turned[4][MINE];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, piece = lane >> 4;
    int e, a, b;
    if (!find_tile(g.offsets, g.E, g.R, g.chunk, blockIdx.x, e, a, b)) return;
    if (e == g.E) {                                            // rows behind the last segment
        constexpr int PIECE = 16 / sizeof(D);
        const int pieces = g.M / PIECE;
        for (int i = threadIdx.x; i < (b - a) * pieces; i += 4 * kWave)
            *reinterpret_cast<u32x4*>(reinterpret_cast<D*>(g.d) + (int64_t)(a + i / pieces) * g.ldd + i % pieces * PIECE) = u32x4{0, 0, 0, 0};
        return;
    }
    char* zt = turned[wave];
    char* xt = zt + 32 * QS * 128;
    u32x4 p[MT][QS];
    narrow_matrix<T, LIN_DX, MT, QS>(g, e, p);
    f32x4 sum[MT][CT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int v = 0; v < CT; ++v) sum[t][v] = f32x4{0.f, 0.f, 0.f, 0.f};
    const char* Q = reinterpret_cast<const char*>(g.q);
    const char* Y = reinterpret_cast<const char*>(g.mask);
    const char* X = reinterpret_cast<const char*>(g.x);
    for (int r0 = a + wave * 64; r0 < b; r0 += 4 * 64) {
        int row = min(r0 + lane, b - 1);                       // of x, one to a lane
        if (g.rows) { row = g.rows[row]; row = row >= 0 ? g.top_k(row) : -1; }
        if (r0 + lane >= b || row >= g.x_rows) row = -1;
        u32x4 q[4][QS], y[MASK ? 4 : 1][MASK ? QS : 1], x[4][XS];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = r0 + u * 16 + c;
#pragma unroll
            for (int s = 0; s < QS; ++s) {
                const int at = s * 32 + piece * 8;
                const bool in = r < b && at < g.K;
                q[u][s] = load16(in ? Q + ((int64_t)r * g.ldq + at) * 2 : zero_row());
                if (MASK) y[u][s] = load16(in ? Y + ((int64_t)r * g.ldmask + at) * 2 : zero_row());
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = __shfl(row, u * 16 + c);
#pragma unroll
            for (int s = 0; s < XS; ++s) {
                const int at = s * 32 + piece * 8;
                x[u][s] = load16(r >= 0 && at < g.M ? X + ((int64_t)r * g.ldx + at) * 2 : zero_row());
            }
        }
        if (MASK)
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int s = 0; s < QS; ++s)
#pragma unroll
                    for (int w = 0; w < 4; ++w) q[u][s][w] = keep_where(q[u][s][w], y[u][s][w]);
        put_turned<QS>(zt, q, 32 * QS);
        put_turned<XS>(xt, x, 16 * MT);
        wave_lds_fence();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            f32x4 acc[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < QS; ++s)
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[t] = mfma16<T>(p[t][s], q[u][s], acc[t]);
            if (r0 + u * 16 + c < b) narrow_store<D, MT>(g, r0 + u * 16 + c, acc, false);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            u32x4 fx[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) fx[t] = *reinterpret_cast<const u32x4*>(xt + turned_at(t * 16 + c, s * 4 + piece));
#pragma unroll
            for (int v = 0; v < CT; ++v) {
                const u32x4 fz = *reinterpret_cast<const u32x4*>(zt + turned_at(v * 16 + c, s * 4 + piece));
#pragma unroll
                for (int t = 0; t < MT; ++t) sum[t][v] = mfma16<T>(fx[t], fz, sum[t][v]);
            }
        }
        wave_lds_fence();
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int v = 0; v < CT; ++v) *reinterpret_cast<f32x4*>(zt + (t * CT + v) * 1024 + lane * 16) = sum[t][v];
    __syncthreads();
    if ((int)blockIdx.x >= g.R / g.chunk + g.E) return;        // (never, of a plan's offsets)
    for (int i = wave; i < MT * CT; i += 4) {
        f32x4 s = *reinterpret_cast<const f32x4*>(turned[0] + i * 1024 + lane * 16);
#pragma unroll
        for (int w = 1; w < 4; ++w) s += *reinterpret_cast<const f32x4*>(turned[w] + i * 1024 + lane * 16);
        const int m = i / CT * 16 + piece * 4, o = i % CT * 16 + c;
        if (m < g.M && o < g.K) *reinterpret_cast<f32x4*>(g.partial + ((int64_t)blockIdx.x * g.K + o) * g.M + m) = s;
    }
}

template <typename T, typename D, int MT, int QS>
static void narrow_bwd_tile(const LinArgs& g, hipStream_t st) {
    const unsigned blocks = (unsigned)(g.R / g.chunk + g.E + 1);
    if (g.mask) expert_narrow_bwd_kernel<T, D, MT, QS, true><<<blocks, 4 * kWave, 0, st>>>(g);
    else expert_narrow_bwd_kernel<T, D, MT, QS, false><<<blocks, 4 * kWave, 0, st>>>(g);
}
template <typename T, typename D, int MT>
static void narrow_bwd_m(const LinArgs& g, hipStream_t st) {
    if (g.K <= 32) narrow_bwd_tile<T, D, MT, 1>(g, st);
    else narrow_bwd_tile<T, D, MT, 2>(g, st);
}
template <typename T, typename D>
static void narrow_bwd(const LinArgs& g, hipStream_t st) {
    if (g.M <= 16) narrow_bwd_m<T, D, 1>(g, st);
    else if (g.M <= 32) narrow_bwd_m<T, D, 2>(g, st);
    else narrow_bwd_m<T, D, 4>(g, st);
}
// rows per chunk where both gradients of a layer are made at once (0: they are not): for three workgroups per CU, as the table above says
static int narrow_bwd_chunk(int64_t R, int n_in, int n_out) {
    if (n_in > 64 || n_out > 64 || R < 8 * NARROW_ROWS) return 0;
    const int64_t chunk = (R / (3 * (int64_t)num_cus()) + NARROW_ROWS) / NARROW_ROWS * NARROW_ROWS;
    return (int)std::min<int64_t>(chunk, 1 << 20);
}

template <typename T, typename D, int MODE, int MT, int QS>
static void narrow_launch_tile(const LinArgs& g, hipStream_t st) {
    const unsigned blocks = (unsigned)(g.R / NARROW_ROWS + g.E + 1);
    constexpr bool MAY_MASK = MODE != LIN_FWD;
    if (MAY_MASK && g.mask) expert_narrow_kernel<T, D, MODE, MT, QS, MAY_MASK><<<blocks, 4 * kWave, 0, st>>>(g);
    else expert_narrow_kernel<T, D, MODE, MT, QS, false><<<blocks, 4 * kWave, 0, st>>>(g);
}
template <typename T, typename D, int MODE, int MT>
static void narrow_launch_m(const LinArgs& g, hipStream_t st) {
    if (g.K <= 32) narrow_launch_tile<T, D, MODE, MT, 1>(g, st);
    else narrow_launch_tile<T, D, MODE, MT, 2>(g, st);
}
template <typename T, typename D, int MODE>
static void narrow_launch(const LinArgs& g, hipStream_t st) {
    if (g.M <= 16) narrow_launch_m<T, D, MODE, 1>(g, st);
    else if (g.M <= 32) narrow_launch_m<T, D, MODE, 2>(g, st);
    else narrow_launch_m<T, D, MODE, 4>(g, st);
}

// dz of the routed rows, once: where many tiles would read y and mask dy again.  Bound by memory: 32768 x 2048, 403 MB: 68 us (5.9 TB/s, partly from the caches).
__global__ __launch_bounds__(256) void expert_mask_kernel(LinArgs g, u32x4* __restrict__ dz) {
    const int pieces = g.K / 8;
    const int64_t all = (int64_t)min(max(g.offsets[g.E], 0), g.R) * pieces;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / pieces;
        const int at = (int)(i - r * pieces) * 16;
        u32x4 v = load16(reinterpret_cast<const char*>(g.q) + r * g.ldq * 2 + at);
        const u32x4 y = load16(reinterpret_cast<const char*>(g.mask) + r * g.ldmask * 2 + at);
#pragma unroll
        for (int w = 0; w < 4; ++w) v[w] = keep_where(v[w], y[w]);
        dz[i] = v;
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------
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
static bool lin_stride(int64_t stride, int n) { return stride >= n && stride % 8 == 0 && stride <= NSX_MAX_EXPERT_STRIDE; }

template <typename T, int MODE, int TM, int TC, int WM, int WC, bool F32>
static int lin_launch_tile(LinArgs g, hipStream_t st) {
    constexpr int lds = std::max((int)lin_rows(TM + TC), WM * WC * 32 * (TM / WM * 2 + 16));
    static_assert(lds <= 65536, "");
    g.m_tiles = (g.M + TM - 1) / TM;
    g.c_tiles = (g.C + TC - 1) / TC;
    int64_t blocks;
    if (MODE == LIN_DW) {
        const int wm = lin_group_dw(g.m_tiles), wc = lin_group_dw(g.c_tiles);
        const int64_t groups = (g.chunk > 0 ? g.R / g.chunk + g.E : g.E) * (int64_t)((g.m_tiles + wm - 1) / wm) * ((g.c_tiles + wc - 1) / wc);
        blocks = (groups + 7) / 8 * 8 * wm * wc;
    } else {
        blocks = ((int64_t)g.R / TC + g.E + 1) * g.m_tiles;
        blocks = (blocks + 7) / 8 * 8;
    }
    NSX_REQUIRE(blocks * (WM * WC * kWave) < ((int64_t)1 << 32), "expert_linear: %lld tiles are more than one launch", (long long)blocks);
    constexpr bool MAY_MASK = MODE != LIN_FWD && TM * TC <= 128 * 128;
    if (MAY_MASK && g.mask) expert_linear_kernel<T, MODE, TM, TC, WM, WC, MAY_MASK, F32><<<(unsigned)blocks, WM * WC * kWave, lds, st>>>(g);
    else expert_linear_kernel<T, MODE, TM, TC, WM, WC, false, F32><<<(unsigned)blocks, WM * WC * kWave, lds, st>>>(g);
    return NSX_OK;
}

// ---- which tile size ----------------------------------------------------------------------------------------------
// Forward and dx, us by (rows x choices of experts, n_in -> n_out), bf16, 64 x 64 | 128 x 128 tiles:
//   4096 x 2 of 16, 1024 -> 1024  39.8 | 34.5      1024 x 2 of 16, 512 -> 512  10.9 | 11.4       4 x 8 of 64, 1024 -> 1024  15.1 | 17.1
//   32 x 8 of 64, 1024 -> 1024    26.7 | 28.4      256 x 8 of 64, 1024 -> 1024 35.9 | 34.8
//   262144 x 2 of 16, 32 -> 64    30.2 | 38.4      262144 x 2 of 16, 64 -> 16  27.1 | 36.2
// The small tile where the result is no wider than it, where a segment has but a few rows, or where the large ones are fewer
// than the CUs.
static bool small_tiles(const LinArgs& g) {
    const int64_t rows = g.R / 128 + std::min<int64_t>(g.E, g.R);
    return g.M <= 64 || g.R < 16 * (int64_t)g.E || rows * ((g.M + 127) / 128) < num_cus();
}
// dW, chunk (0: none) and tile.  us with chunks of 256 | 512 | 1024 | 2048 | 4096 rows, then without:
//   262144 x 2 of 16,  32 ->   64   64 x 64 tiles   37 |  31 |  30 |  40                  128 x 128 tiles   47 |  40 |  39 |  46
//    65536 x 2 of 16, 128 ->  128   64 x 64 tiles   31 |  27 |  30 |  42                  128 x 128 tiles   32 |  28 |  32 |  46
//    65536 x 2 of 16, 256 ->  256   64 x 64 tiles  108 |  88 |  80 |  63 |  87;  247      128 x 128 tiles   93 |  76 |  65 |  60 |  92;  282
//    65536 x 2 of 16, 512 ->  512   64 x 64 tiles    - | 316 | 224 | 199 | 204;  276      128 x 128 tiles    - | 259 | 160 | 141 | 146;  285
//    65536 x 2 of 4, 1024 -> 1024   64 x 64 tiles    - | 998 | 787 | 690 | 646;  761      128 x 128 tiles    - | 834 | 585 | 466 | 402;  800
//    16384 x 2 of 8,  768 ->  768   64 x 64 tiles  250 | 148 | 119 | 111 |   -;  116      128 x 128 tiles  278 | 164 | 129 | 115 |   -;  122
//     8192 x 2 of 16, 512 ->  512   64 x 64 tiles   50 |  40 |  38 |  44 |   -;   35      128 x 128 tiles   46 |  37 |  36 |  44 |   -;   36
//     5003 x 3 of 23, 176 ->  136   64 x 64 tiles   21 |  22 |  27 |  32                  128 x 128 tiles   22 |  24 |  30 |  36
// Short chunks fill the card, long ones keep the partial sums small beside what is read: two workgroups per CU of the large tiles,
// four of the small ones.  Without chunks where the matrices have tiles enough: 16384 x 2 of 16, 1024 -> 2048 then takes 570 | 180;
// of small tiles only up to 8192 rows per expert.  (The lines above have segments of 0.4 to 1.5 of the mean.  Where they are nearly
// equal, both gradients with chunks of large tiles | without chunks, small ones: 16384 x 2 of 8, 768 -> 768  203 | 168;  8192 x 2 of 16,
// 512 -> 512  63 | 53;  65536 x 2 of 16, 512 -> 512  318 | 344;  of 4, 1024 -> 1024  898 | 1110.)
struct DwPlan { int chunk; bool small; };
static DwPlan dw_plan(int64_t R, int E, int n_in, int n_out) {
    const int64_t cus = num_cus();
    const int64_t large = (int64_t)((n_in + 127) / 128) * ((n_out + 127) / 128), small = (int64_t)((n_in + 63) / 64) * ((n_out + 63) / 64);
    if (large * E >= 2 * cus) return {0, false};
    auto rows = [](int64_t n, int64_t least, int64_t most) { return (int)std::min(std::max((n + LIN_BQ - 1) / LIN_BQ * LIN_BQ, least), most); };
    const bool enough = small * E >= 4 * cus;
    if (n_in >= 256 && n_out >= 256 && R * large >= 512 * 2 * cus && (!enough || R >= 8192 * (int64_t)E)) return {rows(R * large / (2 * cus), 512, 4096), false};
    if (enough || R < 8 * (int64_t)LIN_BQ) return {0, true};
    return {rows(R * small / (4 * cus), 4 * LIN_BQ, 1024), true};
}

// The largest products: a wave's tile of 128 x 64 needs three quarters of the LDS reads.  us with 128 x 128 | 256 x 128 | 128 x 256:
//   16384 x 2 of 16, 1024 -> 2048   forward 196 | 181 | 186   dx 174 | 168 | 175   dW 190 | 190 | 168
//   16384 x 2 of 8,  2048 -> 2048   forward 319 | 298 | 310   dx 305 | 309 | 305   dW 355 | 336 | 293
//    8192 x 2 of 16, 1024 -> 1024   forward  52 |  58 |  63   dx  54 |  57 |  62   dW  56 |  65 |  55
//    2048 x 8 of 256, 2048 -> 1024  forward 257 | 243 |       dx 253 | 233     (64 x 64: 269, 276)
// dx of gathered rows, in 32 bits and with the join, 128 x 128 | 256 x 128: first line 240 | 229, second 407 | 415, last 300 | 283.
// As time = f + q s the forward of the first line has f = 36 us (its result's bytes alone 27), s = 133 us per 1024 of q, 1030 TFLOP/s.
// Matrix units busy 37 % of the cycles, LDS 32 %; the rest is the chain of a step (its loads, two barriers, stores, first fragments)
// that two workgroups per CU cover in part: without loads it takes 22 us less, without stores into LDS 30 less again.  256 x 256
// tiles with 4 waves of 128 x 128 have one workgroup per CU, whose start and stores nothing covers: f = 59, the same s; with loads
// straight into LDS each step waits for its memory (1.3 us after the issue at the earliest; the products take 1.2).
// Where segments have a few rows the 64 x 64 tiles stay: 64 x 8 of 256, 1024 -> 2048: forward 150 | 167 (256 x 128), dx 145 | 149.
static bool large_tiles(int64_t tiles128) { return tiles128 >= 6 * (int64_t)num_cus(); }

// dz in a pass of its own (3 R n_out 16-bit values) or masked wherever dy is read (y once more per 128 input features in both
// gradients, registers that large tiles do not have).  us, both gradients, masked in place | once:
//   16384 x 2 of 16, 1024 -> 2048  583 | 454    2048 -> 1024  605 | 470    8192 x 2, 1024 -> 1024  158 | 144    64 x 8 of 64, 1024 -> 1024  92 | 72
//   65536 x 2 of 16,  512 -> 128   263 | 246     256 -> 256   198 | 188    128 -> 128  76 | 79                  4096 x 2, 512 -> 512  49 | 47
static bool mask_once(int64_t R, int n_in, int n_out) { return n_in >= 1024 || (n_in >= 256 && R * n_out >= 1 << 23); }

template <typename T, int MODE, bool F32>
static int lin_launch(const LinArgs& g, bool small, hipStream_t st) {
    if constexpr (MODE != LIN_DW)
        if (g.M <= 64 && g.K <= 64 && (MODE == LIN_FWD || g.M * g.K <= 2048)) {
            narrow_launch<T, std::conditional_t<F32, float, T>, MODE>(g, st);
            return NSX_OK;
        }
    if constexpr (MODE != LIN_DW || !F32)
        if (!g.mask) {                  // (with a mask to apply they do not fit the registers)
            const int64_t tm = (g.M + 127) / 128;
            if constexpr (MODE != LIN_DW) {
                if (!small && g.M > 128 && large_tiles((g.R / 128 + std::min(g.E, g.R)) * tm)) return lin_launch_tile<T, MODE, 256, 128, 2, 2, F32>(g, st);
            } else if (g.C > 128 && large_tiles(g.E * tm * ((g.C + 127) / 128))) return lin_launch_tile<T, MODE, 128, 256, 1, 4, F32>(g, st);
        }
    if (small) return lin_launch_tile<T, MODE, 64, 64, 1, 2, F32>(g, st);
    return lin_launch_tile<T, MODE, 128, 128, 2, 2, F32>(g, st);
}


}  // namespace nsx

extern "C" {

int nsx_expert_linear_fwd(const void* x, int dtype, int64_t x_stride, int64_t x_rows, const int32_t* rows, int top_k,
                          const void* weight, int n_in, int n_out, int E, const int32_t* offsets, int64_t R, int relu, void* y,
                          void* stream) {
    using namespace nsx;
    int rc = lin_check("nsx_expert_linear_fwd", dtype, n_in, n_out, E, R, top_k, offsets);
    if (rc != NSX_OK) return rc;
    if (R == 0) return NSX_OK;
    NSX_REQUIRE(weight && y && (x || x_rows == 0) && aligned16(x) && aligned16(weight) && aligned16(y) && lin_stride(x_stride, n_in),
                "nsx_expert_linear_fwd: NULL or unaligned pointer or row stride %lld", (long long)x_stride);
    NSX_REQUIRE(x_rows >= 0 && x_rows <= NSX_MAX_EXPERT_ENTRIES && (rows || x_rows == R), "nsx_expert_linear_fwd: x has %lld rows", (long long)x_rows);
    LinArgs g{};
    g.p = weight; g.q = x; g.d = y; g.ldp = n_in; g.ldq = x_stride; g.ldd = n_out; g.p_expert = (int64_t)n_in * n_out;
    g.offsets = offsets; g.rows = rows; g.top_k = fast_div(top_k); g.E = E; g.R = (int)R; g.x_rows = (int)x_rows;
    g.M = n_out; g.K = n_in; g.relu = relu;
    rc = dtype == NSX_DTYPE_F16 ? lin_launch<half_t, LIN_FWD, false>(g, small_tiles(g), (hipStream_t)stream)
                                 : lin_launch<bf16_t, LIN_FWD, false>(g, small_tiles(g), (hipStream_t)stream);
    if (rc != NSX_OK) return rc;
    NSX_LAUNCH_CHECK("nsx_expert_linear_fwd");
    return NSX_OK;
}

// workspace: dx in the plan's order, dW's partial sums, masked dy (each a multiple of 16 bytes)
// choices: of a row of x (0: x holds ordered rows).  One choice is rounded once as it is; more are summed in 32 bits.
static int64_t bwd_dx_bytes(int64_t R, int n_in, int choices) { return choices > 0 ? R * n_in * (choices > 1 ? 4 : 2) : 0; }
static int64_t bwd_dw_bytes(int64_t R, int E, int n_in, int n_out, bool with_dx) {
    int chunk = with_dx ? nsx::narrow_bwd_chunk(R, n_in, n_out) : 0;
    if (chunk == 0) chunk = nsx::dw_plan(R, E, n_in, n_out).chunk;
    return chunk > 0 ? (R / chunk + E) * n_in * n_out * 4 : 0;
}
static int64_t bwd_dz_bytes(int64_t R, int n_in, int n_out) { return nsx::mask_once(R, n_in, n_out) ? R * n_out * 2 : 0; }

int64_t nsx_expert_linear_bwd_workspace(int64_t R, int E, int n_in, int n_out, int want_dx, int choices, int want_dw, int masked) {
    using namespace nsx;
    int32_t some = 0;
    const int rc = lin_check("nsx_expert_linear_bwd_workspace", NSX_DTYPE_F16, n_in, n_out, E, R, 1, &some);
    if (rc != NSX_OK) return rc;
    NSX_REQUIRE(choices >= 0 && choices <= NSX_MAX_TOP_K, "nsx_expert_linear_bwd_workspace: %d choices of a row", choices);
    return (want_dx ? bwd_dx_bytes(R, n_in, choices) : 0) + (want_dw ? bwd_dw_bytes(R, E, n_in, n_out, want_dx) : 0) +
           (masked ? bwd_dz_bytes(R, n_in, n_out) : 0);
}

int nsx_expert_linear_bwd(const void* x, int dtype, int64_t x_stride, int64_t x_rows, const int32_t* rows, const int32_t* positions,
                          int top_k, const void* weight, const void* dy, int64_t dy_stride, const void* y, int64_t y_stride, int n_in,
                          int n_out, int E, const int32_t* offsets, int64_t R, void* dx, int dw_f32, void* dw, void* workspace,
                          void* stream) {
    using namespace nsx;
    int rc = lin_check("nsx_expert_linear_bwd", dtype, n_in, n_out, E, R, top_k, offsets);
    if (rc != NSX_OK) return rc;
    NSX_REQUIRE(x_rows >= 0 && x_rows <= NSX_MAX_EXPERT_ENTRIES / top_k && (rows ? x_rows * top_k == R : x_rows == R),
                "nsx_expert_linear_bwd: x has %lld rows", (long long)x_rows);
    NSX_REQUIRE((R == 0 || dy) && aligned16(dy) && aligned16(y) && lin_stride(dy_stride, n_out) && (!y || lin_stride(y_stride, n_out)),
                "nsx_expert_linear_bwd: NULL or unaligned dy or y, or their row strides");
    NSX_REQUIRE(!dx || (aligned16(dx) && (R == 0 || (weight && aligned16(weight) && (!rows || positions)))),
                "nsx_expert_linear_bwd: dx needs aligned pointers, weight and, for gathered rows, positions");
    NSX_REQUIRE(!dw || (aligned16(dw) && (x || x_rows == 0) && aligned16(x) && lin_stride(x_stride, n_in)),
                "nsx_expert_linear_bwd: dw needs aligned pointers and x (row stride %lld)", (long long)x_stride);
    const int64_t dx_bytes = dx ? bwd_dx_bytes(R, n_in, rows ? top_k : 0) : 0, dw_bytes = dw ? bwd_dw_bytes(R, E, n_in, n_out, dx != nullptr) : 0;
    const int64_t dz_bytes = y ? bwd_dz_bytes(R, n_in, n_out) : 0;
    NSX_REQUIRE(dx_bytes + dw_bytes + dz_bytes == 0 || (workspace && aligned16(workspace)), "nsx_expert_linear_bwd: no workspace");
    hipStream_t st = (hipStream_t)stream;
    LinArgs g{};
    g.q = dy; g.mask = y; g.ldq = dy_stride; g.ldmask = y_stride; g.ldd = n_in; g.offsets = offsets; g.top_k = fast_div(top_k);
    g.E = E; g.R = (int)R; g.M = n_in;
    g.rows = rows; g.x_rows = (int)x_rows; g.C = n_out;
    g.partial = reinterpret_cast<float*>((char*)workspace + dx_bytes);
    if (dz_bytes && (dx || dw)) {
        g.K = n_out;
        u32x4* dz = reinterpret_cast<u32x4*>((char*)workspace + dx_bytes + dw_bytes);
        const int64_t blocks = (R * (n_out / 8) + 255) / 256;
        expert_mask_kernel<<<(unsigned)std::min<int64_t>(blocks, 32 * (int64_t)num_cus()), 256, 0, st>>>(g, dz);
        NSX_LAUNCH_CHECK("nsx_expert_linear_bwd");
        g.q = dz; g.ldq = n_out; g.mask = nullptr;
    }
    const int at_once = dx && dw ? narrow_bwd_chunk(R, n_in, n_out) : 0;
    if (dx && R > 0) {
        const bool sums = rows && top_k > 1;
        LinArgs h = g;
        h.p = weight; h.ldp = n_in; h.p_expert = (int64_t)n_in * n_out; h.d = rows ? workspace : dx; h.K = n_out;
        if (at_once) {
            h.x = x; h.ldx = x_stride; h.chunk = at_once;
            if (dtype == NSX_DTYPE_F16) sums ? narrow_bwd<half_t, float>(h, st) : narrow_bwd<half_t, half_t>(h, st);
            else sums ? narrow_bwd<bf16_t, float>(h, st) : narrow_bwd<bf16_t, bf16_t>(h, st);
        } else {
            h.rows = nullptr; h.x_rows = (int)R;
            const bool small = small_tiles(h);
            if (dtype == NSX_DTYPE_F16) rc = sums ? lin_launch<half_t, LIN_DX, true>(h, small, st) : lin_launch<half_t, LIN_DX, false>(h, small, st);
            else rc = sums ? lin_launch<bf16_t, LIN_DX, true>(h, small, st) : lin_launch<bf16_t, LIN_DX, false>(h, small, st);
            if (rc != NSX_OK) return rc;
        }
        NSX_LAUNCH_CHECK("nsx_expert_linear_bwd");
        // A row's choices are summed, and lie between the two launches, in 32 bits: the sum is rounded, not its terms (rounded terms are
        // off by half a step of each, and one beyond the type's range is infinite where the sum is not).
        if (rows) {
            rc = sums ? expert_join_f32((const float*)workspace, R, n_in, positions, x_rows, top_k, dx, dtype, st)
                      : nsx_expert_combine_fwd(workspace, dtype, n_in, R, n_in, nullptr, positions, x_rows, top_k, dx, nullptr, stream);
            if (rc != NSX_OK) return rc;
        }
    }
    if (dw) {
        const DwPlan how = dw_plan(R, E, n_in, n_out);
        g.chunk = at_once ? at_once : how.chunk;
        g.d = dw; g.d_expert = (int64_t)n_in * n_out;
        if (!at_once) {
            const bool f32 = dw_f32 || g.chunk > 0;
            g.p = x; g.ldp = x_stride;
            if (dtype == NSX_DTYPE_F16) rc = f32 ? lin_launch<half_t, LIN_DW, true>(g, how.small, st) : lin_launch<half_t, LIN_DW, false>(g, how.small, st);
            else rc = f32 ? lin_launch<bf16_t, LIN_DW, true>(g, how.small, st) : lin_launch<bf16_t, LIN_DW, false>(g, how.small, st);
            if (rc != NSX_OK) return rc;
            NSX_LAUNCH_CHECK("nsx_expert_linear_bwd");
        }
        if (g.chunk > 0) {
            const int64_t step = R / g.chunk > 8 * (int64_t)E ? 64 : 1024;
            const dim3 grid((unsigned)std::min<int64_t>(((int64_t)n_in * n_out + step - 1) / step, 4096), E);
            if (dw_f32) expert_sum_chunks_kernel<float><<<grid, 256, 0, st>>>(g, (float*)dw);
            else if (dtype == NSX_DTYPE_F16) expert_sum_chunks_kernel<half_t><<<grid, 256, 0, st>>>(g, (half_t*)dw);
            else expert_sum_chunks_kernel<bf16_t><<<grid, 256, 0, st>>>(g, (bf16_t*)dw);
            NSX_LAUNCH_CHECK("nsx_expert_linear_bwd");
        }
    }
    return NSX_OK;
}

}  // extern "C"
