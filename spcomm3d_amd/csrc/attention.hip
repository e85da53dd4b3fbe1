// Attention over a band, forward and backward.  Row i of a sequence at position p sees column c
// when c <= p and (p - c < window or c < sinks):
//   s_ic = scale <q_i, k_c>,  P_ic = exp(s_ic - lse_i),  o_i = sum_c P_ic v_c
//   dV_c = sum_i P_ic dO_i,  dS_ic = P_ic (<dO_i, v_c> - <dO_i, o_i>),
//   dQ_i = scale sum_c dS_ic k_c,  dK_c = scale sum_i dS_ic q_i.
#include "attention.h"
#include "attention_frag.h"

#include <type_traits>

namespace spc3d {
namespace {

constexpr int kThreads = 256;
constexpr int kFewSteps = 2;

// In a block that few steps enter: as selects instead of a branch, masks would cost every step as much
// as its exponentials.
#define KEEP_BRANCH() asm volatile("")

struct Work {
    uint32_t tile, head;
};
// Workgroups go round-robin to the 8 XCDs.  With a multiple of 8 shared heads each XCD takes whole
// shared heads, so that its L2 holds their keys and values once; otherwise in plain order, the
// heads that share keys next to each other in time.
__device__ __forceinline__ Work work_of(uint32_t id, uint32_t ntiles, uint32_t heads, uint32_t kv_heads)
{
    const uint32_t group = heads / kv_heads;
    if (kv_heads % 8 == 0) {
        const uint32_t j = id / 8, per = ntiles * group, r = j % per;
        return {r / group, ((j / per) * 8 + id % 8) * group + r % group};
    }
    return {id / heads, id % heads};
}

// The steps of kKeyStep columns that rows at positions pa .. pb go over: `first` steps from column
// 0 on for the sinks, then those from step `from` on.
struct Steps {
    int first, from, count;
    __device__ __forceinline__ int at(int k) const { return k < first ? k : from + k - first; }
};
__device__ __forceinline__ Steps steps_of(int pa, int pb, int ncols, int window, int sinks)
{
    const int end = min(pb + 1, ncols); // columns seen lie below
    Steps s{0, 0, 0};
    if (end <= 0)
        return s;
    const int step = (int)kKeyStep;
    const int lo = window > pa ? 0 : pa - window + 1;
    s.first = (min(sinks, end) + step - 1) / step;
    s.from = max(lo / step, s.first);
    s.count = s.first + max(0, (end + step - 1) / step - s.from);
    return s;
}

__device__ __forceinline__ bool sees(int p, int c, int window, int sinks)
{
    return c <= p && (p - c < window || c < sinks);
}

template <typename T> __device__ __forceinline__ bool is_finite(T x) { return fabsf((float)x) < __builtin_inff(); }

// ---- forward --------------------------------------------------------------------------------
// Each wavefront owns 16 NQ rows; K and V come through LDS in steps of 64 columns.  S^T = K Q^T
// leaves lane l with row l % 16, so maxima and sums of a row are over the lane's own registers and
// two exchanges, and the probabilities are the right operand of O^T += V^T P^T where they lie.
// Bound by the matrix units and, between their instructions, by the exponentials: 16,384 rows in bfloat16,
// 32 heads of 128 over 8, window 4096: 1.05 ms, 0.92 PFLOP/s (8192^3 product of the library: 1.23).
// Short or few rows are bound by the launch and the chain of steps: 48 rows, 4 heads of 64: 4.4 us.
template <typename T, int DP, int NQ>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void attend_kernel(BandArgs a)
{
    typedef Tile<T, DP> L;
    constexpr int NS = DP / 32, ND = DP / 16, NT = kKeyStep / 16;
    constexpr int kBytes = kKeyStep * L::kRowBytes;
    // Keys, then values, of this step and of the next.  Two arrays and every other step its own
    // code: the compiler then knows that the reads of one do not wait for the loads of the other.
    __shared__ __align__(16) char even[2 * kBytes], odd[2 * kBytes];

    const Work w = work_of(blockIdx.x, a.ntiles, a.heads, a.kv_heads);
    const RowTile t = a.tiles[w.tile];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane & 15, g = lane >> 4;
    const int dim = (int)a.dim, ncols = (int)t.ncols;
    const uint32_t kvh = w.head / (a.heads / a.kv_heads);
    const T *const qp = (const T *)a.q.p + t.row0 * a.q.stride + w.head * dim;
    const T *const kp = (const T *)a.k.p + t.key0 * a.k.stride + kvh * dim;
    const T *const vp = (const T *)a.v.p + t.key0 * a.v.stride + kvh * dim;

    Frag<T> qf[NQ][NS];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = (wave * NQ + n) * 16 + l;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int d = 32 * s + 8 * g;
            qf[n][s] = r < (int)t.nrow && d < dim ? load_frag(qp + r * a.q.stride + d) : zero_frag<T>();
        }
    }
    const Steps st = steps_of(t.pos0, t.pos0 + (int)t.nrow - 1, ncols, a.window, a.sinks);
    const int wa = t.pos0 + wave * NQ * 16, wb = min(wa + NQ * 16, t.pos0 + (int)t.nrow) - 1;
    const float sc = a.scale * kLog2e;
    if (dim < DP) {
        clear_tile<2 * kBytes, kThreads>(even, tid);
        clear_tile<2 * kBytes, kThreads>(odd, tid);
    }
    auto fetch = [&](int k, char *kt) {
        const int c0 = st.at(k) * (int)kKeyStep;
        char *const vt = kt + kBytes;
        const int id = fresh(tid);
        load_tile<T, DP, kKeyStep, kThreads>(kt, kp + c0 * a.k.stride, a.k.stride, ncols - c0, dim, id);
        load_tile<T, DP, kKeyStep, kThreads>(vt, vp + c0 * a.v.stride, a.v.stride, ncols - c0, dim, id);
    };

    f32x4 acc[ND][NQ];
    float m[NQ], sum[NQ];
    // The second pass, if any, is for values that are not finite: 0 x inf would reach rows that do
    // not see them, so steps with hidden pairs take those values one by one.
    auto pass = [&](auto careful) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n] = kNegInf;
            sum[n] = 0.0f;
#pragma unroll
            for (int d = 0; d < ND; ++d)
                acc[d][n] = f32x4{0, 0, 0, 0};
        }
        __syncthreads(); // the tiles are cleared, or read for the last time
        if (st.count > 0)
            fetch(0, even);
        auto step = [&](int k, char *kt, char *next) __attribute__((always_inline)) {
            const int c0 = st.at(k) * (int)kKeyStep;
            char *const vt = kt + kBytes;
            const int lane = fresh(tid & 63), l = lane & 15, g = lane >> 4;
            loads_done();
            __syncthreads();
            if (k + 1 < st.count)
                fetch(k + 1, next);
            const int c9 = c0 + (int)kKeyStep - 1;
            if (wb < c0 || (wa - c9 >= a.window && c0 >= a.sinks))
                return; // nothing here is seen by this wavefront's rows
            const bool whole = c9 <= wa && (wb - c0 < a.window || c9 < a.sinks);

            f32x4 sv[NT][NQ];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
#pragma unroll
                for (int n = 0; n < NQ; ++n)
                    sv[i][n] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const Frag<T> f = L::rows(kt, 16 * i, s, lane);
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
                        sv[i][n] = mma(f, qf[n][s], sv[i][n]);
                }
            }
            if (!whole) {
                KEEP_BRANCH();
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (!sees(wa + 16 * n + l, c0 + 16 * i + 4 * g + j, a.window, a.sinks))
                                sv[i][n][j] = kNegInf;
            }
            float top[NQ];
            bool grown = false;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                top[n] = sv[0][n][0];
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        top[n] = fmaxf(top[n], sv[i][n][j]);
                top[n] = column_max(top[n]) * sc;
                grown |= top[n] > m[n] + kSlack;
            }
            if (__any(grown)) {
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    const float to = fmaxf(m[n], top[n]);
                    const float down = __builtin_amdgcn_exp2f(m[n] - (to == kNegInf ? 0.0f : to));
                    m[n] = to;
                    sum[n] *= down;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        acc[d][n] *= down;
                }
            }
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                // nothing seen yet: exp2(-inf - 0) = 0
                const float less = (m[n] == kNegInf ? 0.0f : m[n]) - WeightShift<T>::value;
                float add = 0.0f;
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[i][n][j], sc, -less));
                        sv[i][n][j] = p;
                        add += p;
                    }
                sum[n] += add;
            }
            const bool one_by_one = careful.value && !whole;
#pragma unroll
            for (int u = 0; u < NT / 2; ++u) {
                Frag<T> pf[NQ];
#pragma unroll
                for (int n = 0; n < NQ; ++n)
                    pf[n] = join<T>(rounded<T>(sv[2 * u][n]), rounded<T>(sv[2 * u + 1][n]));
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    Frag<T> f = L::columns(vt, 32 * u, d, lane);
                    if constexpr (careful.value) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (one_by_one && !is_finite(f[j]))
                                f[j] = (T)0.0f;
                    }
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
                        acc[d][n] = mma(f, pf[n], acc[d][n]);
                }
            }
            if (one_by_one) {
                for (int c = 0; c < (int)kKeyStep; ++c)
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int e = 16 * d + 4 * g + j;
                            const T x = *reinterpret_cast<const T *>(vt + L::at(c, e / L::kVec) +
                                                                     (e % L::kVec) * sizeof(T));
                            if (!is_finite(x)) {
#pragma unroll
                                for (int n = 0; n < NQ; ++n)
                                    if (sees(wa + 16 * n + l, c0 + c, a.window, a.sinks))
                                        acc[d][n][j] += (float)x;
                            }
                        }
            }
        };
        for (int k = 0; k < st.count; k += 2) {
            step(k, even, odd);
            if (k + 1 < st.count)
                step(k + 1, odd, even);
        }
        int bad = 0;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            sum[n] = column_sum(sum[n]);
            const float by = sum[n] == 0.0f ? 0.0f : 1.0f / sum[n];
            const bool mine = (wave * NQ + n) * 16 + l < (int)t.nrow;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                acc[d][n] *= by;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    bad |= mine && !is_finite(acc[d][n][j]);
            }
        }
        return bad;
    };
    if (__syncthreads_or(pass(std::false_type())))
        pass(std::true_type());
    T *const op = (T *)a.o.p + t.row0 * a.o.stride + w.head * dim;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = (wave * NQ + n) * 16 + l;
        if (r >= (int)t.nrow)
            continue;
#pragma unroll
        for (int d = 0; d < ND; ++d)
            if (16 * d + 4 * g < dim)
                store_half<T>(op + r * a.o.stride + 16 * d + 4 * g, acc[d][n]);
        if (a.lse && g == 0)
            a.lse[(uint64_t)(t.row0 + r) * a.heads + w.head] =
                sum[n] == 0.0f ? kNegInf : (m[n] + __log2f(sum[n]) - WeightShift<T>::value) * kLn2;
    }
}

// ---- backward -------------------------------------------------------------------------------
// Two kernels, one over rows (dQ) and one over columns (dK, dV), each with the scores computed
// again: seven products instead of five, but every sum is one workgroup's, in a fixed order,
// without atomics or a panel of partial dQ.  Bound by the matrix units, the exponentials and the reads of
// LDS between them.  8192 rows in bfloat16, 32 heads of 128 over 8, window 1024: dQ 277 us, dK and dV
// 455, forward 217 before them.
template <typename T, int DP, int NQ>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void attend_dq_kernel(BandArgs a)
{
    typedef Tile<T, DP> L;
    constexpr int NS = DP / 32, ND = DP / 16, NT = kKeyStep / 16;
    constexpr int kBytes = kKeyStep * L::kRowBytes;
    // Keys, then values, of this step and of the next.  Two arrays and every other step its own
    // code: the compiler then knows that the reads of one do not wait for the loads of the other.
    __shared__ __align__(16) char even[2 * kBytes], odd[2 * kBytes];

    const Work w = work_of(blockIdx.x, a.ntiles, a.heads, a.kv_heads);
    const RowTile t = a.tiles[w.tile];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane & 15, g = lane >> 4;
    const int dim = (int)a.dim, ncols = (int)t.ncols;
    const uint32_t kvh = w.head / (a.heads / a.kv_heads);
    const T *const qp = (const T *)a.q.p + t.row0 * a.q.stride + w.head * dim;
    const T *const gp = (const T *)a.d_o.p + t.row0 * a.d_o.stride + w.head * dim;
    const T *const op = (const T *)a.o.p + t.row0 * a.o.stride + w.head * dim;
    const T *const kp = (const T *)a.k.p + t.key0 * a.k.stride + kvh * dim;
    const T *const vp = (const T *)a.v.p + t.key0 * a.v.stride + kvh * dim;

    Frag<T> qf[NQ][NS], gf[NQ][NS];
    float lse[NQ], delta[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = (wave * NQ + n) * 16 + l;
        const bool mine = r < (int)t.nrow;
        float dot = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int d = 32 * s + 8 * g;
            const bool in = mine && d < dim;
            qf[n][s] = in ? load_frag(qp + r * a.q.stride + d) : zero_frag<T>();
            gf[n][s] = in ? load_frag(gp + r * a.d_o.stride + d) : zero_frag<T>();
            const Frag<T> of = in ? load_frag(op + r * a.o.stride + d) : zero_frag<T>();
#pragma unroll
            for (int j = 0; j < 8; ++j)
                dot = __builtin_fmaf((float)gf[n][s][j], (float)of[j], dot);
        }
        delta[n] = column_sum(dot);
        lse[n] = mine ? a.lse[(uint64_t)(t.row0 + r) * a.heads + w.head] * kLog2e : kNegInf;
        if (lse[n] == kNegInf)
            lse[n] = -kNegInf; // a row that sees nothing: every weight is exp2(-inf)
    }
    const Steps st = steps_of(t.pos0, t.pos0 + (int)t.nrow - 1, ncols, a.window, a.sinks);
    const int wa = t.pos0 + wave * NQ * 16, wb = min(wa + NQ * 16, t.pos0 + (int)t.nrow) - 1;
    const float sc = a.scale * kLog2e;
    if (dim < DP) {
        clear_tile<2 * kBytes, kThreads>(even, tid);
        clear_tile<2 * kBytes, kThreads>(odd, tid);
    }
    auto fetch = [&](int k, char *kt) {
        const int c0 = st.at(k) * (int)kKeyStep;
        char *const vt = kt + kBytes;
        const int id = fresh(tid);
        load_tile<T, DP, kKeyStep, kThreads>(kt, kp + c0 * a.k.stride, a.k.stride, ncols - c0, dim, id);
        load_tile<T, DP, kKeyStep, kThreads>(vt, vp + c0 * a.v.stride, a.v.stride, ncols - c0, dim, id);
    };

    f32x4 acc[ND][NQ];
    float weighed[NQ]; // sum of P dP: <dO, o> again, without the rounding of o
    // Rows that see few columns take it before they use it: their dS is a small difference, and
    // the rounding of o in <dO, o> would show (dQ of 300 rows in bfloat16: 1.72 times the error of
    // one rounding, 1.47 so; further down the sequence it is lost among the columns).
    auto pass = [&](auto last) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            weighed[n] = 0.0f;
#pragma unroll
            for (int d = 0; d < ND; ++d)
                acc[d][n] = f32x4{0, 0, 0, 0};
        }
        __syncthreads(); // the tiles are cleared, or read for the last time
        if (st.count > 0)
            fetch(0, even);
        auto step = [&](int k, char *kt, char *next) __attribute__((always_inline)) {
            const int c0 = st.at(k) * (int)kKeyStep;
            char *const vt = kt + kBytes;
            const int lane = fresh(tid & 63), l = lane & 15, g = lane >> 4;
            loads_done();
            __syncthreads();
            if (k + 1 < st.count)
                fetch(k + 1, next);
            const int c9 = c0 + (int)kKeyStep - 1;
            if (wb < c0 || (wa - c9 >= a.window && c0 >= a.sinks))
                return;
            const bool whole = c9 <= wa && (wb - c0 < a.window || c9 < a.sinks);
#pragma unroll
            for (int u = 0; u < NT / 2; ++u) {
                HalfFrag<T> ds[2][NQ];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    f32x4 sv[NQ], dp[NQ];
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
                        sv[n] = dp[n] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < NS; ++s) {
                        const Frag<T> f = L::rows(kt, 32 * u + 16 * i, s, lane);
                        const Frag<T> h = L::rows(vt, 32 * u + 16 * i, s, lane);
#pragma unroll
                        for (int n = 0; n < NQ; ++n) {
                            sv[n] = mma(f, qf[n][s], sv[n]);
                            dp[n] = mma(h, gf[n][s], dp[n]);
                        }
                    }
                    if (!whole) {
                KEEP_BRANCH();
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (!sees(wa + 16 * n + l, c0 + 32 * u + 16 * i + 4 * g + j, a.window, a.sinks)) {
                                    sv[n][j] = kNegInf;
                                    dp[n][j] = 0.0f;
                                }
                    }
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[n][j], sc, -lse[n]));
                            weighed[n] = __builtin_fmaf(p, dp[n][j], weighed[n]);
                            sv[n][j] = p * (dp[n][j] - delta[n]);
                        }
                        ds[i][n] = rounded<T>(sv[n]);
                    }
                }
                if constexpr (last.value) {
                    Frag<T> df[NQ];
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
                        df[n] = join<T>(ds[0][n], ds[1][n]);
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const Frag<T> f = L::columns(kt, 32 * u, d, lane);
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
                            acc[d][n] = mma(f, df[n], acc[d][n]);
                    }
                }
            }
        };
        for (int k = 0; k < st.count; k += 2) {
            step(k, even, odd);
            if (k + 1 < st.count)
                step(k + 1, odd, even);
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n)
            delta[n] = column_sum(weighed[n]);
    };
    if (st.count <= kFewSteps)
        pass(std::false_type());
    pass(std::true_type());
    T *const dqp = (T *)a.dq.p + t.row0 * a.dq.stride + w.head * dim;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        const int r = (wave * NQ + n) * 16 + l;
        if (r >= (int)t.nrow)
            continue;
#pragma unroll
        for (int d = 0; d < ND; ++d)
            if (16 * d + 4 * g < dim)
                store_half<T>(dqp + r * a.dq.stride + 16 * d + 4 * g, acc[d][n] * a.scale);
        if (g == 0) {
            const uint64_t at = (uint64_t)(t.row0 + r) * a.heads + w.head;
            a.stats[at] = lse[n];
            a.stats[a.nstats + at] = delta[n];
        }
    }
    if (blockIdx.x == 0 && tid == 0) { // what rows past a tile's end read
        a.stats[a.nstats - 1] = -kNegInf;
        a.stats[2 * a.nstats - 1] = 0.0f;
    }
}

// Each wavefront owns 32 columns of the tile's 128, whose keys and values stay in its registers
// (values of the largest heads in LDS: two wavefronts to a SIMD have room for the sums, the keys and
// some fragments ahead, and no more);
// rows (of every head that shares them) come through LDS 64 (32) at a time.  S = Q K^T leaves a lane
// with one column and the rows 4 g + i, 16 + 4 g + i, which is the left operand of dV += P^T dO and
// dK += dS^T Q as it lies.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 2 : 1) void attend_dkv_kernel(BandArgs a)
{
    typedef Tile<T, DP> L;
    constexpr int NS = DP / 32, ND = DP / 16, NK = 2;
    constexpr bool kKeepV = dkv_keeps_v(sizeof(T), DP);
    constexpr int ROWS = dkv_row_step(sizeof(T), DP);
    constexpr float kUp = sizeof(T) == 2 && WeightShift<T>::value != 0 ? 32768.0f : 1.0f; // weights are at most 1 here
    constexpr int kBytes = ROWS * L::kRowBytes;
    // Q, then dO, then lse and <dO, o> of the rows
    __shared__ __align__(16) char even[2 * kBytes + 8 * ROWS], odd[2 * kBytes + 8 * ROWS];
    __shared__ __align__(16) char values[kKeepV ? 16 : kKeyTile * L::kRowBytes];

    const uint32_t group = a.heads / a.kv_heads;
    const Work w = work_of(blockIdx.x, a.npieces, a.kv_heads, a.kv_heads);
    const KeyPiece t = a.pieces[w.tile];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane & 15, g = lane >> 4;
    const int dim = (int)a.dim, nrow = (int)t.nrow;
    const T *const kp = (const T *)a.k.p + t.key0 * a.k.stride + w.head * dim;
    const T *const vp = (const T *)a.v.p + t.key0 * a.v.stride + w.head * dim;

    Frag<T> kf[NK][NS], vf[NK][kKeepV ? NS : 1];
    f32x4 dk[NK][ND], dv[NK][ND];
#pragma unroll
    for (int n = 0; n < NK; ++n) {
        const int r = ((t.spread ? 0 : wave * NK) + n) * 16 + l;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int d = 32 * s + 8 * g;
            const bool in = r < (int)t.nkey && d < dim;
            kf[n][s] = in ? load_frag(kp + r * a.k.stride + d) : zero_frag<T>();
            if constexpr (kKeepV)
                vf[n][s] = in ? load_frag(vp + r * a.v.stride + d) : zero_frag<T>();
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
            dk[n][d] = dv[n][d] = f32x4{0, 0, 0, 0};
    }
    const int wave_first = t.spread ? 0 : wave * NK * 16; // its first column
    const int ca = t.col0 + wave_first, cb = ca + (t.spread ? (int)kSpread : NK * 16) - 1;
    const float sc = a.scale * kLog2e;
    const int per = (nrow + ROWS - 1) / ROWS, first = (int)t.step0, end = first + (int)t.nsteps;

    if (dim < DP) {
        clear_tile<2 * kBytes, kThreads>(even, tid);
        clear_tile<2 * kBytes, kThreads>(odd, tid);
        if constexpr (!kKeepV) {
            clear_tile<kKeyTile * L::kRowBytes, kThreads>(values, tid);
            __syncthreads();
        }
    }
    if constexpr (!kKeepV)
        if (first < end) // no load may outlive its workgroup
            load_tile<T, DP, kKeyTile, kThreads>(values, vp, a.v.stride, (int)t.nkey, dim, tid);
    auto fetch = [&](int k, char *qt) {
        char *const gt = qt + kBytes;
        const uint32_t head = w.head * group + k / per;
        const int r0 = (k % per) * ROWS;
        const uint64_t row = t.row0 + r0;
        const int id = fresh(tid);
        load_tile<T, DP, ROWS, kThreads>(qt, (const T *)a.q.p + row * a.q.stride + head * dim, a.q.stride, nrow - r0,
                                         dim, id);
        load_tile<T, DP, ROWS, kThreads>(gt, (const T *)a.d_o.p + row * a.d_o.stride + head * dim, a.d_o.stride,
                                         nrow - r0, dim, id);
        const int part = __builtin_amdgcn_readfirstlane(id >> 6);
        if (part * 64 < 2 * ROWS) { // rows past the end weigh nothing
            const int r = id % ROWS;
            const uint64_t at = r0 + r < nrow ? (row + r) * a.heads + head : a.nstats - 1;
            __builtin_amdgcn_global_load_lds((global_void *)(a.stats + id / ROWS * a.nstats + at),
                                             (lds_void *)(gt + kBytes + part * 256), 4, 0, 0);
        }
    };
    __syncthreads();
    if (first < end)
        fetch(first, even);
    // A piece of the sinks: every wavefront has the same 16 columns (n = 0) and sums its own
    // quarter of the elements, dk[0][d] then being element 16 (wave kQuarter + d) + l.
    constexpr int kQuarter = (ND + 3) / 4;
    auto step = [&](auto spread, int k, char *qt, char *next) __attribute__((always_inline)) {
        constexpr int NK = spread.value ? 1 : 2;
        char *const gt = qt + kBytes;
        const float *const stat = (const float *)(gt + kBytes);
        const int lane = fresh(tid & 63), l = lane & 15, g = lane >> 4;
        loads_done();
        __syncthreads();
        if (k + 1 < end)
            fetch(k + 1, next);
        const int pa = t.pos0 + (k % per) * ROWS, pb = pa + ROWS - 1;
        if (pb < ca || (pa - cb >= a.window && ca >= a.sinks))
            return;
        const bool whole = pa >= cb && (pb - ca < a.window || cb < a.sinks);

#pragma unroll
        for (int u = 0; u < ROWS / 32; ++u) {
            HalfFrag<T> ps[2][NK], ds[2][NK];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f32x4 sv[NK], dp[NK];
#pragma unroll
                for (int n = 0; n < NK; ++n)
                    sv[n] = dp[n] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    const Frag<T> f = L::rows(qt, 32 * u + 16 * i, s, lane);
                    const Frag<T> h = L::rows(gt, 32 * u + 16 * i, s, lane);
#pragma unroll
                    for (int n = 0; n < NK; ++n) {
                        sv[n] = mma(f, kf[n][s], sv[n]);
                        dp[n] = mma(h, kKeepV ? vf[n][kKeepV ? s : 0] : L::rows(values, wave_first + 16 * n, s, lane),
                                    dp[n]);
                    }
                }
                const f32x4 lse = *reinterpret_cast<const f32x4 *>(stat + 32 * u + 16 * i + 4 * g);
                const f32x4 delta = *reinterpret_cast<const f32x4 *>(stat + ROWS + 32 * u + 16 * i + 4 * g);
                if (!whole) {
                KEEP_BRANCH();
#pragma unroll
                    for (int n = 0; n < NK; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (!sees(pa + 32 * u + 16 * i + 4 * g + j, ca + 16 * n + l, a.window, a.sinks)) {
                                sv[n][j] = kNegInf;
                                dp[n][j] = 0.0f;
                            }
                }
#pragma unroll
                for (int n = 0; n < NK; ++n) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[n][j], sc, -lse[j]));
                        sv[n][j] = p * kUp;
                        dp[n][j] = p * (dp[n][j] - delta[j]);
                    }
                    ps[i][n] = rounded<T>(sv[n]);
                    ds[i][n] = rounded<T>(dp[n]);
                }
            }
            Frag<T> pf[NK], df[NK];
#pragma unroll
            for (int n = 0; n < NK; ++n) {
                pf[n] = join<T>(ps[0][n], ps[1][n]);
                df[n] = join<T>(ds[0][n], ds[1][n]);
            }
#pragma unroll
            for (int d = 0; d < (spread.value ? kQuarter : ND); ++d) {
                const int dd = spread.value ? wave * kQuarter + d : d;
                // (a quarter past the last element takes that one again: nobody reads its sums)
                const Frag<T> f = L::columns(gt, 32 * u, spread.value ? min(dd, ND - 1) : dd, lane);
                const Frag<T> h = L::columns(qt, 32 * u, spread.value ? min(dd, ND - 1) : dd, lane);
#pragma unroll
                for (int n = 0; n < NK; ++n) {
                    dv[n][d] = mma(pf[n], f, dv[n][d]);
                    dk[n][d] = mma(df[n], h, dk[n][d]);
                }
            }
        }
    };
    auto walk = [&](auto spread) __attribute__((always_inline)) {
        for (int k = first; k < end; k += 2) {
            step(spread, k, even, odd);
            if (k + 1 < end)
                step(spread, k + 1, odd, even);
        }
    };
    if (t.spread)
        walk(std::true_type());
    else
        walk(std::false_type());
    // lane l holds element 16 d + l of the columns 4 g + j
    T *const dkp = (T *)a.dk.p + t.key0 * a.dk.stride + w.head * dim;
    T *const dvp = (T *)a.dv.p + t.key0 * a.dv.stride + w.head * dim;
    float *const part = t.slot == kNoSlot
                            ? nullptr
                            : a.partial + ((uint64_t)t.slot * a.kv_heads + w.head) * 2 * kKeyTile * dim;
    if (t.spread) {
#pragma unroll
        for (int d = 0; d < kQuarter; ++d)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = 4 * g + j, e = 16 * (wave * kQuarter + d) + l;
                if (c < (int)t.nkey && e < dim) {
                    part[c * dim + e] = dk[0][d][j];
                    part[(kKeyTile + c) * dim + e] = dv[0][d][j] * (1.0f / kUp);
                }
            }
        return;
    }
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = (wave * NK + n) * 16 + 4 * g + j;
            if (c >= (int)t.nkey)
                continue;
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const int e = 16 * d + l;
                if (e >= dim)
                    continue;
                if (part) {
                    part[c * dim + e] = dk[n][d][j];
                    part[(kKeyTile + c) * dim + e] = dv[n][d][j] * (1.0f / kUp);
                } else {
                    dkp[c * a.dk.stride + e] = (T)(dk[n][d][j] * a.scale);
                    dvp[c * a.dv.stride + e] = (T)(dv[n][d][j] * (1.0f / kUp));
                }
            }
        }
}

// The pieces of a tile of columns joined in their order.  Bound by the chain of loads of one element's
// pieces, so four elements a lane and four pieces at a time: 5 us for the sinks of 8192 rows, 5 and 10 us where
// every tile is cut (1000 rows in single precision; 6000 in bfloat16), where one element and piece took 6, 13 and 12.
template <typename T> __global__ __launch_bounds__(kThreads) void join_dkv_kernel(BandArgs a)
{
    const KeySplit t = a.splits[blockIdx.x];
    const uint32_t h = blockIdx.y, dim = a.dim;
    const uint64_t step = (uint64_t)a.kv_heads * 2 * kKeyTile * dim;
    const float *const part = a.partial + ((uint64_t)t.first * a.kv_heads + h) * 2 * kKeyTile * dim;
    const uint32_t i = (blockIdx.z * kThreads + threadIdx.x) * 4;
    if (i >= t.nkey * dim)
        return;
    const uint32_t c = i / dim, e = i % dim, n = t.count + (c < kSpread ? t.spread : 0);
    f32x4 x = {}, y = {};
    uint32_t s = 0;
    for (; s + 4 <= n; s += 4) {
        f32x4 u[4], w[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            u[j] = *(const f32x4 *)(part + (s + j) * step + i);
            w[j] = *(const f32x4 *)(part + (s + j) * step + kKeyTile * dim + i);
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            x += u[j];
            y += w[j];
        }
    }
    for (; s < n; ++s) {
        x += *(const f32x4 *)(part + s * step + i);
        y += *(const f32x4 *)(part + s * step + kKeyTile * dim + i);
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) {
        ((T *)a.dk.p)[(t.key0 + c) * a.dk.stride + h * dim + e + j] = (T)(x[j] * a.scale);
        ((T *)a.dv.p)[(t.key0 + c) * a.dv.stride + h * dim + e + j] = (T)y[j];
    }
}

__global__ __launch_bounds__(kThreads) void fill_short_kernel(int dtype, void *p, uint64_t n, float value)
{
    const bf16_t b = (bf16_t)value;
    const f16_t h = (f16_t)value;
    const uint16_t w = dtype == 2 ? __builtin_bit_cast(uint16_t, b) : __builtin_bit_cast(uint16_t, h);
    for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (uint64_t)gridDim.x * kThreads)
        if (dtype == 4)
            ((uint8_t *)p)[i] = to_f8(value);
        else
            ((uint16_t *)p)[i] = w;
}

enum class Op { kForward, kDq, kDkv };

template <typename T, int DP> void launch_one(const BandArgs &a, Op op, uint32_t tile_rows, hipStream_t s)
{
    const dim3 block(kThreads), rows(a.ntiles * a.heads);
    if (op == Op::kDkv)
        hipLaunchKernelGGL((attend_dkv_kernel<T, DP>), dim3(a.npieces * a.kv_heads), block, 0, s, a);
    else if (op == Op::kDq && tile_rows == 128)
        hipLaunchKernelGGL((attend_dq_kernel<T, DP, 2>), rows, block, 0, s, a);
    else if (op == Op::kDq)
        hipLaunchKernelGGL((attend_dq_kernel<T, DP, 1>), rows, block, 0, s, a);
    else if (tile_rows == 128)
        hipLaunchKernelGGL((attend_kernel<T, DP, 2>), rows, block, 0, s, a);
    else
        hipLaunchKernelGGL((attend_kernel<T, DP, 1>), rows, block, 0, s, a);
}

hipError_t launch(const BandArgs &a, Op op, uint32_t tile_rows, hipStream_t s)
{
    const int dp = (int)padded_dim(a.dtype == 0 ? 4 : 2, a.dim);
    switch (a.dtype * 1000 + dp) {
    case 64: launch_one<float, 64>(a, op, tile_rows, s); break;
    case 128: launch_one<float, 128>(a, op, tile_rows, s); break;
    case 2064: launch_one<bf16_t, 64>(a, op, tile_rows, s); break;
    case 2096: launch_one<bf16_t, 96>(a, op, tile_rows, s); break;
    case 2128: launch_one<bf16_t, 128>(a, op, tile_rows, s); break;
    case 3064: launch_one<f16_t, 64>(a, op, tile_rows, s); break;
    case 3096: launch_one<f16_t, 96>(a, op, tile_rows, s); break;
    case 3128: launch_one<f16_t, 128>(a, op, tile_rows, s); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

} // namespace

hipError_t launch_attend(const BandArgs &a, uint32_t tile_rows, hipStream_t stream)
{
    return a.ntiles ? launch(a, Op::kForward, tile_rows, stream) : hipSuccess;
}

hipError_t launch_attend_dq(const BandArgs &a, uint32_t tile_rows, hipStream_t stream)
{
    return a.ntiles ? launch(a, Op::kDq, tile_rows, stream) : hipSuccess;
}

hipError_t launch_attend_dkv(const BandArgs &a, hipStream_t stream)
{
    if (!a.npieces)
        return hipSuccess;
    hipError_t e = launch(a, Op::kDkv, 0, stream);
    if (e != hipSuccess || !a.nsplits)
        return e;
    const dim3 grid(a.nsplits, a.kv_heads, (kKeyTile * a.dim + 4 * kThreads - 1) / (4 * kThreads));
    switch (a.dtype) {
    case 0: hipLaunchKernelGGL((join_dkv_kernel<float>), grid, dim3(kThreads), 0, stream, a); break;
    case 2: hipLaunchKernelGGL((join_dkv_kernel<bf16_t>), grid, dim3(kThreads), 0, stream, a); break;
    default: hipLaunchKernelGGL((join_dkv_kernel<f16_t>), grid, dim3(kThreads), 0, stream, a); break;
    }
    return hipGetLastError();
}

hipError_t launch_fill_short(int dtype, void *p, uint64_t n, float value, hipStream_t stream)
{
    if (n == 0)
        return hipSuccess;
    const uint32_t grid = (uint32_t)((n + kThreads - 1) / kThreads < 4096 ? (n + kThreads - 1) / kThreads : 4096);
    hipLaunchKernelGGL(fill_short_kernel, dim3(grid), dim3(kThreads), 0, stream, dtype, p, n, value);
    return hipGetLastError();
}

uint64_t partial_floats(uint32_t nslots, uint32_t kv_heads, uint32_t dim)
{
    return (uint64_t)nslots * kv_heads * 2 * kKeyTile * dim;
}

} // namespace spc3d
