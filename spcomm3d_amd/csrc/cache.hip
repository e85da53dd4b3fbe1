// A paged cache of keys and values: new rows put into it, rotated and rounded on the way, and
// attention of a few rows over it.
#include "cache.h"
#include "attention_frag.h"

#include <type_traits>

namespace spc3d {
namespace {

constexpr int kThreads = 256;

// What a sequence is, with nothing past what the caller's bounds allow.
struct Seq {
    uint32_t row0, n; // its rows
    int len, first;   // tokens held; position of row row0 (negative: len is less than n)
};
__device__ __forceinline__ Seq seq_of(const SeqsView &s, uint32_t b, uint32_t page)
{
    Seq q;
    q.row0 = min(s.starts[b], s.rows);
    q.n = min(max(min(s.starts[b + 1], s.rows), q.row0) - q.row0, s.max_rows);
    q.len = (int)min(min((uint64_t)s.lens[b], (uint64_t)s.max_len), (uint64_t)s.table_stride * page);
    q.first = q.len - (int)q.n;
    return q;
}

// ---- append -----------------------------------------------------------------------------------
// What rotates eight elements of a head, from d on: cosines and sines of their angles, and where the other
// one of each pair (j, j + turned / 2) is.
struct Turn {
    f32x8 cos, sin;
    int other; // element of the other; negative: nothing to rotate
    float sign;
};
__device__ __forceinline__ Turn turn_of(const float *rotations, int turned, int64_t pos, int d)
{
    Turn t;
    t.other = -1;
    if (rotations && d < turned) {
        const int half = turned / 2, at = d < half ? d : d - half;
        const float *const c = rotations + pos * turned + at;
        t.cos = load_frag(c);
        t.sin = load_frag(c + half);
        t.other = d < half ? d + half : at;
        t.sign = d < half ? -1.0f : 1.0f;
    }
    return t;
}
// Eight elements from d on of the row at `p`, rotated.  Products and sums are rounded one by one, as the
// formula is written.
template <typename T> __device__ __forceinline__ f32x8 rotated(const T *p, int d, const Turn &t)
{
#pragma clang fp contract(off)
    const Frag<T> x = load_frag(p + d);
    f32x8 y;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        y[j] = (float)x[j];
    if (t.other >= 0) {
        const Frag<T> z = load_frag(p + t.other);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            y[j] = y[j] * t.cos[j] + t.sign * ((float)z[j] * t.sin[j]);
    }
    return y;
}
template <typename T>
__device__ __forceinline__ f32x8 rotated(const T *p, int d, const float *rotations, int turned, int64_t pos)
{
    return rotated(p, d, turn_of(rotations, turned, pos, d));
}

// The smallest 2^e, -40 <= e <= 40, with most <= 448 * 2^e.
__device__ __forceinline__ float scale_for(float most)
{
    const uint32_t bits = __float_as_uint(most);
    const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
    return __uint_as_float((uint32_t)(min(max(e, -40), 40) + 127) << 23);
}

__device__ __forceinline__ u32x2 pack_f8(const float *x)
{
    u32x2 w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        int v = __builtin_amdgcn_cvt_pk_fp8_f32(f8_range(x[4 * h]), f8_range(x[4 * h + 1]), 0, false);
        w[h] = __builtin_amdgcn_cvt_pk_fp8_f32(f8_range(x[4 * h + 2]), f8_range(x[4 * h + 3]), v, true);
    }
    return w;
}
__device__ __forceinline__ void unpack_f8(u32x2 w, float *x)
{
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
        x[4 * h] = a[0];
        x[4 * h + 1] = a[1];
        x[4 * h + 2] = b[0];
        x[4 * h + 3] = b[1];
    }
}

// One workgroup has the keys or the values of one page and head to itself, so that a page's scale
// and the re-rounding of what it holds need no other's word.  C: what the cache holds.
template <typename T, typename C>
__device__ __forceinline__ void append_page(const AppendArgs &a, uint32_t b, uint32_t nth, uint32_t head, bool values,
                                            float *reduce, T *tile)
{
    constexpr bool kF8 = sizeof(C) == 1;
    const Seq s = seq_of(a.s, b, a.c.page);
    const int page = (int)a.c.page, dim = (int)a.c.dim, tid = threadIdx.x;
    const int begin = max(s.first, 0);
    if (!s.n || begin >= s.len)
        return;
    const int p = begin / page + (int)nth;
    const int lo = max(begin - p * page, 0), hi = min(s.len - p * page, page); // new slots
    if (lo >= hi)
        return;
    const uint32_t id = a.s.table[(uint64_t)b * a.s.table_stride + p];
    if (id >= a.c.npages)
        return;
    const uint64_t unit = (uint64_t)id * a.c.heads + head;
    const HeadsView &from = values ? a.v : a.k;
    const T *const src = (const T *)from.p + head * dim;
    C *const dst = (C *)(values ? a.c.v : a.c.k) + unit * page * dim;
    const float *const rot = values ? nullptr : a.rotations;
    // panel row of slot j: row0 + (p page + j - first)
    const int64_t row0 = (int64_t)s.row0 + (int64_t)p * page - s.first;
    const int chunks = dim / 8, wide = dim + 8;

    // Values come by row and go by element, through LDS: 16 bytes a lane either way.
    if (values && !kF8)
        for (int i = tid; i < (hi - lo) * chunks; i += kThreads) {
            const int j = lo + i / chunks, d = i % chunks * 8;
            *(Frag<T> *)(tile + j * wide + d) = load_frag(src + (row0 + j) * from.stride + d);
        }
    float scale = 1.0f, ratio = 1.0f;
    if constexpr (kF8) {
        float most = 0.0f;
        for (int i = tid; i < (hi - lo) * chunks; i += kThreads) {
            const int j = lo + i / chunks, d = i % chunks * 8;
            const f32x8 x = rotated(src + (row0 + j) * from.stride, d, rot, (int)a.turned, (int64_t)p * page + j);
            if (values)
                *(Frag<T> *)(tile + j * wide + d) = load_frag(src + (row0 + j) * from.stride + d);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (fabsf(x[e]) < __builtin_inff())
                    most = fmaxf(most, fabsf(x[e]));
        }
#pragma unroll
        for (int m = 32; m; m >>= 1)
            most = fmaxf(most, __shfl_xor(most, m));
        if ((tid & 63) == 0)
            reduce[tid >> 6] = most;
        float *const held = (values ? a.c.v_scale : a.c.k_scale) + unit;
        const float before = *held;
        __syncthreads();
        scale = scale_for(fmaxf(fmaxf(reduce[0], reduce[1]), fmaxf(reduce[2], reduce[3])));
        if (lo > 0) { // the page was begun before
            const float held_by = before > 0 ? before : 0.0f;
            scale = fmaxf(scale, held_by);
            ratio = held_by / scale;
        }
        if (tid == 0)
            *held = scale; // every thread has read it
    }
    const int from_slot = ratio == 1.0f ? lo : 0; // a larger scale: what the page holds is rounded again
    if (!values) {
        for (int i = tid; i < (hi - from_slot) * chunks; i += kThreads) {
            const int j = from_slot + i / chunks, d = i % chunks * 8;
            C *const to = dst + j * dim + d;
            float x[8];
            if constexpr (kF8) {
                if (j < lo) {
                    unpack_f8(*(const u32x2 *)to, x);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[e] *= ratio;
                } else {
                    const f32x8 y = rotated(src + (row0 + j) * from.stride, d, rot, (int)a.turned, (int64_t)p * page + j);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[e] = y[e] / scale;
                }
                *(u32x2 *)to = pack_f8(x);
            } else {
                const f32x8 y = rotated(src + (row0 + j) * from.stride, d, rot, (int)a.turned, (int64_t)p * page + j);
                Frag<C> f;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    f[e] = (C)y[e];
                *(Frag<C> *)to = f;
            }
        }
        return;
    }
    if (!kF8)
        __syncthreads(); // (8 bits: there was one since the tile was written)
    // eight slots of one element at a time, the slots of an element next to each other
    const int first = from_slot / 8, blocks = (hi + 7) / 8 - first;
    for (int i = tid; i < blocks * dim; i += kThreads) {
        const int d = i / blocks, j0 = (first + i - d * blocks) * 8;
        C *const to = dst + (uint64_t)d * page + j0;
        const bool all = j0 >= lo && j0 + 8 <= hi; // nothing of what was there stays
        T x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            x[e] = all || (j0 + e >= lo && j0 + e < hi) ? tile[(j0 + e) * wide + d] : (T)0.0f;
        if constexpr (kF8) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[e] = (float)x[e] / scale;
            u32x2 was = {0, 0};
            if (!all) {
                float old[8];
                was = *(const u32x2 *)to;
                unpack_f8(was, old);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (j0 + e < lo)
                        y[e] = old[e] * ratio;
            }
            u32x2 w = pack_f8(y);
            if (j0 + 8 > hi) { // slots that no token has yet keep what they hold
                const int keep = hi - j0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int n = min(max(keep - 4 * h, 0), 4);
                    const uint32_t mask = n == 4 ? 0xffffffffu : (1u << 8 * n) - 1;
                    w[h] = (w[h] & mask) | (was[h] & ~mask);
                }
            }
            *(u32x2 *)to = w;
        } else {
            Frag<C> f = zero_frag<C>();
            if (!all)
                f = *(const Frag<C> *)to;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (all || (j0 + e >= lo && j0 + e < hi))
                    f[e] = (C)x[e];
            *(Frag<C> *)to = f;
        }
    }
}

// The sequence that a row belongs to: the last one that starts at or before it and is not empty.
__device__ __forceinline__ uint32_t seq_of_row(const SeqsView &s, uint32_t row)
{
    uint32_t lo = 0, hi = s.nseq; // starts[lo] <= row < starts[hi], where starts ascend
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (s.starts[mid] <= row)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// A row of queries, rotated by `lanes` of which this is number `lane`: one keeps its place in a head from one load to the next where heads
// divide them, and its angles with it.
template <typename T> __device__ __forceinline__ void turn_queries(const AppendArgs &a, uint32_t row, int lane, int lanes)
{
    const uint32_t b = seq_of_row(a.s, row);
    const Seq s = seq_of(a.s, b, a.c.page);
    if (row < s.row0 || row - s.row0 >= s.n)
        return;
    const int pos = s.first + (int)(row - s.row0), dim = (int)a.c.dim, chunks = dim / 8, all = (int)a.q_heads * chunks;
    const float *const rotations = pos < 0 ? nullptr : a.rotations;
    const T *const src = (const T *)a.q.p + row * a.q.stride;
    T *const dst = (T *)a.q_out.p + row * a.q_out.stride;
    const int ahead = lanes / chunks, more = lanes % chunks; // heads and chunks from one load to the next
    int h = lane / chunks, c = lane % chunks;
    Turn t = turn_of(rotations, (int)a.turned, pos, c * 8);
#pragma unroll 4
    for (int i = lane; i < all; i += lanes) {
        if (more)
            t = turn_of(rotations, (int)a.turned, pos, c * 8);
        const f32x8 y = rotated(src + h * dim, c * 8, t);
        Frag<T> f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            f[e] = (T)y[e];
        *(Frag<T> *)(dst + h * dim + c * 8) = f;
        h += ahead;
        c += more;
        if (c >= chunks) {
            c -= chunks;
            ++h;
        }
    }
}

// Workgroups: first those of pages, a.each heads of a page's keys or values each, then those of queries, a.rows_each
// rows each.
// Bound by memory when there are many rows (8 sequences of 1777 in bfloat16, 32 heads of 128 over 8: 76 us,
// 4.6 TB/s), by the launch and the chain page, scale, row, code otherwise (64 rows in 8 bits: 6.7 us).
template <typename T, typename C> __global__ __launch_bounds__(kThreads) void append_kernel(AppendArgs a, uint32_t per_seq)
{
    __shared__ float reduce[kThreads / 64];
    extern __shared__ __align__(16) char tile[]; // page rows of dim + 8 elements
    const uint32_t parts = (a.c.heads + a.each - 1) / a.each, pages = a.s.nseq * per_seq * parts * 2;
    uint32_t id = blockIdx.x;
    if (id >= pages) {
        const uint32_t lanes = kThreads / a.rows_each;
        const uint32_t row = (id - pages) * a.rows_each + __builtin_amdgcn_readfirstlane(threadIdx.x / lanes);
        if (row < a.s.rows)
            turn_queries<T>(a, row, (int)(threadIdx.x % lanes), (int)lanes);
        return;
    }
    const bool values = id & 1;
    id >>= 1;
    const uint32_t first = id % parts * a.each, end = min(first + a.each, a.c.heads);
    id /= parts;
    for (uint32_t head = first; head < end; ++head) {
        if (head > first)
            __syncthreads(); // the last head's maxima and values are read
        append_page<T, C>(a, id / per_seq, id % per_seq, head, values, reduce, (T *)tile);
    }
}

// ---- read -------------------------------------------------------------------------------------
// Columns are the (row, head) pairs that share a kv head, 16 NC of them a workgroup; its four
// wavefronts take the steps of its share of the tokens in turn, each with its own running maximum and sum, joined
// at the end.  Nothing goes through LDS on the way: S^T = K Q^T wants a token's elements, O^T =
// V^T P^T an element's tokens, and that is how the cache holds them.  A lane loads 16 bytes, so a
// step has 4 kTok tokens, kTok of them (16 in 8 bits, 8 in 16) in a group of lanes.  Which token stands
// in which row of S^T is free; they are dealt so that a lane's weights are the tokens kTok g ..
// of its own group, which is what it loads of V.
// What bounds it is memory: K of the next step is asked for as soon as K of this one is used, V
// likewise, so that a wavefront has 8 to 16 KiB under way at any time.  4 sequences of 90,001 to
// 110,000 tokens in 8 bits, 8 heads of 128: 152 us, 5.4 TB/s; 64 of 200 to 4000: 38 us, 4.5 TB/s;
// 16 times 5 rows that see 1000 tokens in half precision: 16 us, 2.1 TB/s (few steps, bound by their chain).
template <typename T> __device__ __forceinline__ Frag<T> from_f8(uint32_t lo, uint32_t hi);
template <> __device__ __forceinline__ bf16x8 from_f8<bf16_t>(uint32_t lo, uint32_t hi)
{
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const auto c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
template <> __device__ __forceinline__ f16x8 from_f8<f16_t>(uint32_t lo, uint32_t hi)
{
    typedef uint32_t u32;
    const u32 a = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
    const u32 b = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
    const u32 c = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
    const u32 d = __builtin_bit_cast(u32, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
    return __builtin_bit_cast(f16x8, u32x4{a, b, c, d});
}

__device__ __forceinline__ bool sees(int p, int c, int window, int sinks)
{
    return c <= p && (p - c < window || c < sinks);
}

// Steps of `size` tokens that rows at positions pa .. pb go over (see attention.hip).
struct Steps {
    int first, from, count;
    __device__ __forceinline__ int at(int k) const { return k < first ? k : from + k - first; }
};
__device__ __forceinline__ Steps steps_of(int pa, int pb, int len, int window, int sinks, int size)
{
    const int end = min(pb + 1, len);
    Steps s{0, 0, 0};
    if (end <= 0)
        return s;
    const int lo = window > pa ? 0 : pa - window + 1;
    s.first = (min(sinks, end) + size - 1) / size;
    s.from = max(lo / size, s.first);
    s.count = s.first + max(0, (end + size - 1) / size - s.from);
    return s;
}

// A row and head's sums over some tokens, in a workspace of dim + 4 floats: maximum (base 2), sum of
// weights, 2 unused, sums of values.
// ONE: a row for each sequence.  Its heads all see the same tokens.
template <typename T, typename C, int DP, int NC, bool ONE>
__global__ __launch_bounds__(kThreads, ONE && NC == 1 && (sizeof(C) == 2 || DP == 64) ? 3 : 2) void read_kernel(ReadArgs a)
{
    constexpr bool kF8 = sizeof(C) == 1;
    constexpr int NS = DP / 32, ND = DP / 16, COLS = 16 * NC;
    constexpr int kTok = 16 / (int)sizeof(C), kStep = 4 * kTok, NT = kTok / 4, KL = DP / (4 * kTok);
    __shared__ float out[4][COLS][DP + 4]; // by wavefront; 4 more: no two columns on the same banks
    __shared__ float part_m[4][COLS], part_sum[4][COLS];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane & 15, g = lane >> 4;
    const int dim = (int)a.c.dim, page = (int)a.c.page, shift = __builtin_ctz(a.c.page);
    const uint32_t group = a.heads / a.c.heads;
    uint32_t id = blockIdx.x;
    const uint32_t head = id % a.c.heads;
    id /= a.c.heads;
    // first shares first: those that short sequences do not have come last, when slots are free
    const uint32_t tile = id % a.col_tiles;
    id /= a.col_tiles;
    const uint32_t b = id % a.s.nseq, split = id / a.s.nseq;
    const Seq s = seq_of(a.s, b, a.c.page);
    const int cols = (int)(s.n * group), m0 = (int)tile * COLS;
    if (m0 >= cols)
        return;
    const int pa = s.first + m0 / (int)group, pb = s.first + (min(m0 + COLS, cols) - 1) / (int)group;
    const Steps st = steps_of(pa, pb, a.c.npages ? s.len : 0, a.window, a.sinks, kStep);
    // every share but the last has a.share steps
    const int k0 = (int)min((uint64_t)split * a.share, (uint64_t)st.count);
    const int k1 = split + 1 == a.splits ? st.count : min(k0 + (int)a.share, st.count);
    if (k0 >= k1 && a.splits > 1) { // no tokens for this share
        if (tid < COLS && m0 + tid < cols) {
            const int mm = m0 + tid;
            const uint64_t row = s.row0 + mm / (int)group;
            float *const to = a.partial + ((row * a.heads + head * group + mm % (int)group) * a.splits + split) * (dim + 4);
            to[0] = kNegInf;
            to[1] = 0.0f;
        }
        return;
    }

    Frag<T> qf[NC][NS];
    int pos[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        const int m = m0 + 16 * n + l, i = m / (int)group, h = (int)head * (int)group + m % (int)group;
        pos[n] = m < cols ? s.first + i : -1;
        const T *const qp = (const T *)a.q.p + (s.row0 + i) * a.q.stride + h * dim;
#pragma unroll
        for (int t = 0; t < NS; ++t) {
            const int d = kF8 ? 64 * (t / 2) + 16 * g + 8 * (t % 2) : 32 * t + 8 * g;
            qf[n][t] = m < cols && d < dim ? load_frag(qp + d) : zero_frag<T>();
        }
    }
    const uint32_t *const table = a.s.table + (uint64_t)b * a.s.table_stride;
    const float sc = a.scale * kLog2e;

    // Pages of the tokens that a lane loads keys of, and values of, in step k; tokens that are not
    // there are loaded from page 0 and hidden.
    struct Pages {
        uint32_t k, v;
    };
    auto pages_of = [&](int k) __attribute__((always_inline)) {
        const int c0 = st.at(k) * kStep, ck = c0 + kTok * (l >> 2), cv = c0 + kTok * g;
        return Pages{ck < s.len ? table[ck >> shift] : a.c.npages, cv < s.len ? table[cv >> shift] : a.c.npages};
    };
    u32x4 kr[NT][KL], vr[ND];
    float k_scale = 1.0f, v_scale = 1.0f;
    bool there = false; // the page of this lane's values
    auto load_k = [&](int k, const Pages &p) __attribute__((always_inline)) {
        const int lane = fresh(tid & 63), l = lane & 15, g = lane >> 4;
        const int ck = st.at(k) * kStep + kTok * (l >> 2);
        const C *kp = (const C *)a.c.k + (((uint64_t)(p.k < a.c.npages ? p.k : 0) * a.c.heads + head) * page +
                                          (ck & (page - 1)) + (l & 3)) * dim;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
#pragma unroll
            for (int t = 0; t < KL; ++t) // elements past the head's are met by zeros of q
                kr[i][t] = *(const u32x4 *)(kp + min(t * 4 * kTok + g * kTok, dim - kTok));
            kp = fresh(kp + 4 * dim); // one address, not all at once
        }
    };
    auto load_v = [&](int k, const Pages &p) __attribute__((always_inline)) {
        const int lane = fresh(tid & 63), l = lane & 15, g = lane >> 4;
        const int cv = st.at(k) * kStep + kTok * g;
        const uint64_t unit = (uint64_t)(p.v < a.c.npages ? p.v : 0) * a.c.heads + head;
        const C *const vp = (const C *)a.c.v + unit * page * dim + (cv & (page - 1));
#pragma unroll
        for (int d = 0; d < ND; ++d) // sums of elements past the head's are not stored
            vr[d] = *(const u32x4 *)(vp + min(16 * d + l, dim - 1) * page);
    };
    auto load_scales = [&](const Pages &p) __attribute__((always_inline)) {
        there = p.v < a.c.npages;
        if constexpr (kF8) {
            const uint64_t unit = (uint64_t)(there ? p.v : 0) * a.c.heads + head;
            k_scale = a.c.k_scale[unit];
            v_scale = a.c.v_scale[unit];
        }
    };

    f32x4 acc[ND][NC];
    float m[NC], sum[NC], ref;
    // Values that are not finite reach rows that do not see them as 0 x inf: such a result is
    // computed once more, carefully (see attend_kernel).
    auto pass = [&](auto careful) __attribute__((always_inline)) {
        ref = 0.0f;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
            m[n] = kNegInf;
            sum[n] = 0.0f;
#pragma unroll
            for (int d = 0; d < ND; ++d)
                acc[d][n] = f32x4{0, 0, 0, 0};
        }
        int k = k0 + wave;
        if (k >= k1)
            return false;
        Pages next = pages_of(k);
        load_k(k, next);
        load_scales(next);
        load_v(k, next);
        auto step = [&](auto more) __attribute__((always_inline)) {
            const int c0 = st.at(k) * kStep, c9 = c0 + kStep - 1, cg = c0 + kTok * g;
            const bool in_v = there;
            float ks = sc * k_scale, vs = v_scale;
            if constexpr (more.value)
                next = pages_of(k + 4);
            f32x4 sv[NT][NC];
#pragma unroll
            for (int i = 0; i < NT; ++i) {
#pragma unroll
                for (int n = 0; n < NC; ++n)
                    sv[i][n] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < NS; ++t) {
                    Frag<T> f;
                    if constexpr (kF8)
                        f = from_f8<T>(kr[i][t / 2][2 * (t % 2)], kr[i][t / 2][2 * (t % 2) + 1]);
                    else
                        f = __builtin_bit_cast(Frag<T>, kr[i][t]);
#pragma unroll
                    for (int n = 0; n < NC; ++n)
                        sv[i][n] = mma(f, qf[n][t], sv[i][n]);
                }
                if constexpr (DP > 64 && (kF8 || NC > 1)) // not every tile's keys widened at once
                    __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (more.value) {
                load_k(k + 4, next);
                load_scales(next);
            }
            // Tokens that no row of the tile sees (not there yet, left of the window) may hold
            // anything: their values become 0.  Edges only, all else is a whole step.
            const bool whole = c9 <= pa && (pb - c0 < a.window || c9 < a.sinks) && __all(in_v);
            if (!whole) {
                asm volatile(""); // a branch, not selects
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t mask = 0;
#pragma unroll
                    for (int e = 0; e < kTok / 4; ++e) {
                        const int c = cg + w * (kTok / 4) + e;
                        const bool seen = in_v && c <= pb && (c < a.sinks || pa - c < a.window);
                        mask |= seen ? (kF8 ? 0xffu << 8 * e : 0xffffu << 16 * e) : 0;
                    }
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        vr[d][w] &= mask;
                }
                if (!in_v || cg > pb || !(cg < a.sinks || pa - (cg + kTok - 1) < a.window))
                    ks = vs = 0.0f; // a scale that belongs to nothing seen
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int n = 0; n < NC; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (in_v && sees(ONE ? pa : pos[n], cg + 4 * i + j, a.window, a.sinks))
                                sv[i][n][j] *= ks;
                            else
                                sv[i][n][j] = kNegInf;
                ks = 1.0f;
            }
            // acc is in units of the largest scale of values so far
            float to_ref = 1.0f, weigh = 1.0f;
            if constexpr (kF8) {
                const float top = fmaxf(ref, column_max(fabsf(vs)));
                to_ref = top > 0 ? ref / top : 0.0f;
                weigh = top > 0 ? vs / top : vs;
                ref = top;
            }
            float top[NC];
            bool grown = kF8 && to_ref != 1.0f;
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                top[n] = kNegInf;
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        sv[i][n][j] *= ks;
                        top[n] = fmaxf(top[n], sv[i][n][j]);
                    }
                top[n] = column_max(top[n]);
                grown |= top[n] > m[n] + kSlack;
            }
            if (__any(grown)) {
#pragma unroll
                for (int n = 0; n < NC; ++n) {
                    const float to = fmaxf(m[n], top[n]);
                    const float down = __builtin_amdgcn_exp2f(m[n] - (to == kNegInf ? 0.0f : to));
                    m[n] = to;
                    sum[n] *= down;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        acc[d][n] *= kF8 ? down * to_ref : down;
                }
            }
#pragma unroll
            for (int n = 0; n < NC; ++n) {
                const float less = (m[n] == kNegInf ? 0.0f : m[n]) - WeightShift<T>::value;
                float add = 0.0f;
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float p = __builtin_amdgcn_exp2f(sv[i][n][j] - less);
                        add += p;
                        sv[i][n][j] = kF8 ? p * weigh : p;
                    }
                sum[n] += add;
            }
#pragma unroll
            for (int u = 0; u < NT / 2; ++u) {
                Frag<T> pf[NC];
#pragma unroll
                for (int n = 0; n < NC; ++n)
                    pf[n] = join<T>(rounded<T>(sv[2 * u][n]), rounded<T>(sv[2 * u + 1][n]));
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    Frag<T> f;
                    if constexpr (kF8)
                        f = from_f8<T>(vr[d][2 * u], vr[d][2 * u + 1]);
                    else
                        f = __builtin_bit_cast(Frag<T>, vr[d]);
                    if constexpr (careful.value) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (!whole && !(fabsf((float)f[j]) < __builtin_inff()))
                                f[j] = (T)0.0f;
                    }
#pragma unroll
                    for (int n = 0; n < NC; ++n)
                        acc[d][n] = mma(f, pf[n], acc[d][n]);
                    if constexpr (DP > 64 && (kF8 || NC > 1))
                        if (d % 2 == 1)
                            __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (careful.value) {
                if (!whole)
                    for (int c = c0; c <= min(c9, pb); ++c) {
                        const uint32_t pc = table[c >> shift];
                        if (pc >= a.c.npages)
                            continue;
                        const C *const from = (const C *)a.c.v + ((uint64_t)pc * a.c.heads + head) * page * dim + (c & (page - 1));
#pragma unroll
                        for (int d = 0; d < ND; ++d)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int e = min(16 * d + 4 * g + j, dim - 1);
                                asm volatile("" ::: "memory"); // one at a time: registers matter here, not time
                                float y;
                                if constexpr (kF8)
                                    y = __builtin_amdgcn_cvt_pk_f32_fp8((int)from[e * page], false)[0];
                                else
                                    y = (float)from[e * page];
                                if (fabsf(y) < __builtin_inff())
                                    continue;
#pragma unroll
                                for (int n = 0; n < NC; ++n)
                                    if (sees(pos[n], c, a.window, a.sinks))
                                        acc[d][n][j] += y;
                            }
                    }
            }
            if constexpr (more.value)
                load_v(k + 4, next);
            k += 4;
        };
        while (k + 4 < k1)
            step(std::true_type());
        step(std::false_type());
        bool bad = false;
        if constexpr (ONE)
            return bad; // no value is hidden from one and seen by another
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    bad |= pos[n] >= 0 && !(fabsf(acc[d][n][j]) < __builtin_inff());
        return (bool)__any(bad);
    };
    if (pass(std::false_type()))
        if constexpr (!ONE)
            pass(std::true_type());

    // the four wavefronts joined, in their order
#pragma unroll
    for (int n = 0; n < NC; ++n) {
        sum[n] = column_sum(sum[n]);
        if (g == 0) {
            part_m[wave][16 * n + l] = m[n];
            part_sum[wave][16 * n + l] = sum[n];
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
            *(f32x4 *)&out[wave][16 * n + l][16 * d + 4 * g] = kF8 ? acc[d][n] * ref : acc[d][n];
    }
    __syncthreads();
    constexpr int kQuads = DP / 4;
    for (int i = tid; i < COLS * kQuads; i += kThreads) {
        const int c = i / kQuads, d = i % kQuads * 4, mm = m0 + c;
        if (mm >= cols || d >= dim)
            continue;
        float top = part_m[0][c];
#pragma unroll
        for (int w = 1; w < 4; ++w)
            top = fmaxf(top, part_m[w][c]);
        const float base = top == kNegInf ? 0.0f : top;
        float total = 0.0f;
        f32x4 y = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float by = __builtin_amdgcn_exp2f(part_m[w][c] - base);
            total += part_sum[w][c] * by;
            y += *(const f32x4 *)&out[w][c][d] * by;
        }
        const uint64_t row = s.row0 + mm / (int)group;
        const uint32_t h = head * group + mm % (int)group;
        if (a.splits > 1) {
            float *const to = a.partial + ((row * a.heads + h) * a.splits + split) * (dim + 4);
            *(f32x4 *)(to + 4 + d) = y;
            if (d == 0) {
                to[0] = top;
                to[1] = total;
            }
        } else {
            const float by = total == 0.0f ? 0.0f : 1.0f / total;
            store_half<T>((T *)a.o.p + row * a.o.stride + h * dim + d, y * by);
            if (d == 0 && a.lse)
                a.lse[row * a.heads + h] = total == 0.0f ? kNegInf : (top + __log2f(total) - WeightShift<T>::value) * kLn2;
        }
    }
}

// The shares of a row and head joined: 32 lanes for its elements, WAYS such groups that take every
// WAYS-th share and are then added in their order.  Bound by its launch and one chain of loads: 5 to 9 us.
template <typename T, int WAYS> __global__ __launch_bounds__(kThreads) void read_join_kernel(ReadArgs a)
{
    constexpr int kRows = kThreads / (32 * WAYS);
    __shared__ float sums[kRows][WAYS][32][5];
    const uint32_t lane = threadIdx.x & 31, way = threadIdx.x / 32 % WAYS, mine = threadIdx.x / (32 * WAYS), dim = a.c.dim;
    const uint64_t at = (uint64_t)blockIdx.x * kRows + mine, row = at / a.heads;
    const uint32_t h = (uint32_t)(at % a.heads);
    bool there = at < (uint64_t)a.s.rows * a.heads;
    if (there) {
        const Seq s = seq_of(a.s, seq_of_row(a.s, (uint32_t)row), a.c.page);
        there = row >= s.row0 && row - s.row0 < s.n;
    }
    const float *const part = a.partial + at * a.splits * (dim + 4);
    float top = kNegInf;
    if (there)
        for (uint32_t i = lane; i < a.splits; i += 32)
            top = fmaxf(top, part[i * (uint64_t)(dim + 4)]);
#pragma unroll
    for (int x = 16; x; x >>= 1)
        top = fmaxf(top, __shfl_xor(top, x));
    const float base = top == kNegInf ? 0.0f : top;
    float total = 0.0f;
    f32x4 y = {0, 0, 0, 0};
    if (there) {
#pragma unroll 4
        for (uint32_t i = way; i < a.splits; i += WAYS) {
            const float *const p = part + i * (uint64_t)(dim + 4);
            if (p[0] == kNegInf)
                continue; // nothing seen in this share, or no tokens: no sums either
            const float by = __builtin_amdgcn_exp2f(p[0] - base);
            total += p[1] * by;
            if (4 * lane < dim)
                y += *(const f32x4 *)(p + 4 + 4 * lane) * by;
        }
    }
    if constexpr (WAYS > 1) {
        float *const to = sums[mine][way][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            to[j] = y[j];
        to[4] = total;
        __syncthreads();
        if (way)
            return;
#pragma unroll
        for (int w = 1; w < WAYS; ++w) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                y[j] += sums[mine][w][lane][j];
            total += sums[mine][w][lane][4];
        }
    }
    if (!there)
        return;
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    if (4 * lane < dim)
        store_half<T>((T *)a.o.p + row * a.o.stride + h * dim + 4 * lane, y * by);
    if (lane == 0 && a.lse)
        a.lse[at] = total == 0.0f ? kNegInf : (top + __log2f(total) - WeightShift<T>::value) * kLn2;
}

template <typename T, typename C, int DP> hipError_t launch_read_one(const ReadArgs &a, hipStream_t s)
{
    const dim3 grid(a.s.nseq * a.col_tiles * a.splits * a.c.heads), block(kThreads);
    const bool narrow = read_columns(a.s.max_rows, a.heads / a.c.heads) == 16;
    if (a.s.max_rows == 1 && narrow)
        hipLaunchKernelGGL((read_kernel<T, C, DP, 1, true>), grid, block, 0, s, a);
    else if (a.s.max_rows == 1)
        hipLaunchKernelGGL((read_kernel<T, C, DP, 2, true>), grid, block, 0, s, a);
    else if (narrow)
        hipLaunchKernelGGL((read_kernel<T, C, DP, 1, false>), grid, block, 0, s, a);
    else
        hipLaunchKernelGGL((read_kernel<T, C, DP, 2, false>), grid, block, 0, s, a);
    const uint64_t rows = (uint64_t)a.s.rows * a.heads;
    if (a.splits > 8)
        hipLaunchKernelGGL((read_join_kernel<T, 8>), dim3((uint32_t)rows), block, 0, s, a);
    else if (a.splits > 1)
        hipLaunchKernelGGL((read_join_kernel<T, 1>), dim3((uint32_t)((rows + 7) / 8)), block, 0, s, a);
    return hipGetLastError();
}

template <typename T> hipError_t launch_read(const ReadArgs &a, hipStream_t s)
{
    if (a.c.dtype == 4)
        return a.c.dim <= 64 ? launch_read_one<T, uint8_t, 64>(a, s) : launch_read_one<T, uint8_t, 128>(a, s);
    return a.c.dim <= 64 ? launch_read_one<T, T, 64>(a, s) : launch_read_one<T, T, 128>(a, s);
}

template <typename T> hipError_t launch_append(const AppendArgs &a, hipStream_t s)
{
    const uint32_t per_seq = (a.s.max_rows + a.c.page - 2) / a.c.page + 1; // pages that so many rows touch
    const uint32_t parts = (a.c.heads + a.each - 1) / a.each, lds = a.c.page * (a.c.dim + 8) * sizeof(T);
    const uint64_t grid = (uint64_t)a.s.nseq * per_seq * parts * 2 + (a.q.p ? (a.s.rows + a.rows_each - 1) / a.rows_each : 0);
    if (a.c.dtype == 4)
        hipLaunchKernelGGL((append_kernel<T, uint8_t>), dim3((uint32_t)grid), dim3(kThreads), lds, s, a, per_seq);
    else
        hipLaunchKernelGGL((append_kernel<T, T>), dim3((uint32_t)grid), dim3(kThreads), lds, s, a, per_seq);
    return hipGetLastError();
}

} // namespace

uint32_t read_columns(uint32_t max_rows, uint32_t group) { return (uint64_t)max_rows * group <= 16 ? 16 : 32; }
uint32_t read_step(int cache_dtype) { return cache_dtype == 4 ? 64 : 32; }

hipError_t launch_cache_append(const AppendArgs &a, hipStream_t stream)
{
    if (!a.s.nseq || !a.s.rows || !a.s.max_rows)
        return hipSuccess;
    return a.dtype == 2 ? launch_append<bf16_t>(a, stream) : launch_append<f16_t>(a, stream);
}

hipError_t launch_cache_read(const ReadArgs &a, hipStream_t stream)
{
    if (!a.s.nseq || !a.s.rows || !a.s.max_rows)
        return hipSuccess;
    return a.dtype == 2 ? launch_read<bf16_t>(a, stream) : launch_read<f16_t>(a, stream);
}

} // namespace spc3d
