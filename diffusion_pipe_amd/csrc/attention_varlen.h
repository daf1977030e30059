// attention_varlen.h -- what the bf16 (attention_varlen.hip) and the fp32 (attention_varlen_f32.hip) kernels of attention over packed sequences share: the arguments, how a workgroup finds
// its sequence, rows and keys, and the kernels that join the parts of a split axis.
#pragma once
#include "dpipe_common.h"

namespace dpipe_varlen {
using namespace dpipe;

struct VarlenShape {
    const int *cu_q, *cu_k;
    float *lse, *delta;                  // [Hq][Tq]
    float *part, *part_lse;              // split forms: forward rows [split][Tq][Hq][D] and their lse [split][Hq][Tq]; dQ [split][Tq][Hq][D], then dK / dV [split][2][Tk][Hk][D]
    long tq, tk;
    int n, hq, hk, g, nsplit, dq_split, causal;
    long q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, do_ss, do_sh;    // o, dq, dk, dv are contiguous
    float scale;
};
template <typename T> struct VarlenParams : VarlenShape {
    const T *q, *k, *v, *dout;
    T *o, *o_lo, *dq, *dk, *dv;          // o_lo (bf16): what the rounding of o left, rounded: o + o_lo is the output to 2^-17, which the backward's delta is formed from
};

constexpr int NT = 256, ROWS = 128;       // threads, query rows (dK / dV: keys) of a workgroup: 4 waves of 32
constexpr float M_INIT = -3.0e38f;       // running maximum before the first key: finite, so that exp2(-inf - m) is 0 and never NaN
constexpr int SORTED = 32;               // sequences up to which their tiles are ordered by work (a forward of 1311 + 2560 + 4608 tokens as packed 378 us, ordered 347; 64 sequences of 128
                                         // tokens 47 as packed, 72 ordered: the order costs a workgroup up to 90 ns a sequence)
constexpr float RESCALE_AT = 8.f;        // the accumulator is rescaled when the maximum grew by more than 2^8: P stays below 256, its relative rounding is the same

// ------------------------------------------------------------------------------------------------ which sequence, which rows
struct Tile { long row0, rows, q0, k0; int lq, lk; bool live; };

// offset i of the ascending sums, kept inside the tensor (i > n: its end)
__device__ __forceinline__ int bound(const int* cu, int i, int n, int total) {
    if (i == 0) return 0;
    if (i > n) return total;
    const int c = cu[i];
    return c < 0 ? 0 : c > total ? total : c;
}
// slot -> sequence and first row; PER = rows per tile, gg = rows per token on the tiled side.  Up to SORTED sequences (a lane each): the tiles of the sequences with the longest other
// side first -- the workgroups with the most work start first -- each sequence's tiles from its ascending sum on, the rows behind the last sequence (n) after them.  More sequences:
// the slots from  start / PER + b  on, in order.  `reversed`: the last tile of a sequence (causal: the one that sees most) first.
template <int PER>
__device__ __forceinline__ Tile find_tile(const VarlenShape& p, int slot, bool keys, bool reversed) {
    const int *cu = keys ? p.cu_k : p.cu_q, *cu2 = keys ? p.cu_q : p.cu_k;
    const int total = (int)(keys ? p.tk : p.tq), total2 = (int)(keys ? p.tq : p.tk), n = p.n;
    const int gg = keys ? 1 : p.g, lane = threadIdx.x & 63;
    int b, at, s0, s1, o0 = 0, o1 = 0;   // sequence, tile of it, its range on the tiled side and on the other (the rows behind the last sequence have no other side)
    if (n <= SORTED) {
        const int i0 = min(lane, n - 1);
        const int my_s0 = bound(cu, i0, n, total), my_s1 = max(my_s0, bound(cu, i0 + 1, n, total)), my_o0 = bound(cu2, i0, n, total2), my_o1 = max(my_o0, bound(cu2, i0 + 1, n, total2));
        const int nt = lane < n ? ((my_s1 - my_s0) * gg + PER - 1) / PER : 0, work = my_o1 - my_o0;
        int start = 0, all = 0;
#pragma unroll 8
        for (int i = 0; i < ((n + 7) & ~7); ++i) {             // (lanes from n on hold no tiles)
            const int nt_i = __builtin_amdgcn_readlane(nt, i), work_i = __builtin_amdgcn_readlane(work, i);
            start += nt_i & -(int)((work_i > work) | ((work_i == work) & (i < lane)));
            all += nt_i;
        }
        const unsigned long long here = __ballot(lane < n && slot >= start && slot < start + nt);
        b = here ? __builtin_amdgcn_readfirstlane(__builtin_ctzll(here)) : n - 1;
        s0 = __builtin_amdgcn_readlane(my_s0, b); s1 = __builtin_amdgcn_readlane(my_s1, b);
        if (here) { at = slot - __builtin_amdgcn_readlane(start, b); o0 = __builtin_amdgcn_readlane(my_o0, b); o1 = __builtin_amdgcn_readlane(my_o1, b); }
        else { at = slot - all; b = n; s0 = s1; s1 = max(s0, total); }
    } else {
        int count = 0;
        for (int base = 0; base <= n; base += 64) {
            const int i = base + lane;
            const int c = __popcll(__ballot(i <= n && (long)bound(cu, i, n, total) * gg / PER + i <= slot));
            count += c;
            if (c < 64) break;
        }
        b = __builtin_amdgcn_readfirstlane(count - 1);
        s0 = bound(cu, b, n, total); s1 = max(s0, bound(cu, b + 1, n, total));
        at = slot - (int)((long)s0 * gg / PER + b);
        if (b < n) { o0 = bound(cu2, b, n, total2); o1 = max(o0, bound(cu2, b + 1, n, total2)); }
    }
    Tile t;
    t.rows = (long)(s1 - s0) * gg;
    const int nt = (int)((t.rows + PER - 1) / PER);
    t.live = at >= 0 && at < nt;         // (offsets that do not ascend reach no row outside their tensor)
    t.row0 = (long)(reversed ? nt - 1 - at : at) * PER;
    t.q0 = keys ? o0 : s0; t.k0 = keys ? s0 : o0;
    t.lq = keys ? o1 - o0 : s1 - s0; t.lk = keys ? s1 - s0 : o1 - o0;
    if (keys && p.causal && t.lq > t.lk) { t.q0 += t.lq - t.lk; t.lq = t.lk; }      // (dK / dV) the queries in front see no key: not read, what they hold is 0 * NaN to nobody
    return t;
}

// The lane's query row: token (in the buffer) and query head; `last`: the last key of its sequence it sees (-1: none)
struct Row { long token, head; int last; bool live; };
__device__ __forceinline__ Row find_row(const VarlenShape& p, const Tile& t, int kh, int wid, int i) {
    const long at = t.row0 + 32 * wid + i;
    Row r;
    r.live = at < t.rows;
    const unsigned row = r.live ? (unsigned)at : 0u, tok = row / (unsigned)p.g;
    r.token = t.q0 + tok; r.head = (long)kh * p.g + (row - tok * p.g);
    r.last = p.causal ? (int)min((long)tok + t.lk - t.lq, (long)t.lk - 1) : t.lk - 1;
    return r;
}
// How many keys (from the first on) some row of the workgroup sees, some row of the wave, every live row of the wave
struct Seen { int group, wave, all; };
__device__ __forceinline__ Seen keys_seen(const VarlenShape& p, const Tile& t, int wid) {
    const long r0 = t.row0 + 32 * wid, last = min(t.row0 + ROWS, t.rows) - 1, wlast = min(r0 + 32, t.rows) - 1;
    if (!p.causal) return {t.lk, wlast < r0 ? 0 : t.lk, t.lk};
    auto upto = [&](long row) { return (int)max(0l, min((long)t.lk, row / p.g + t.lk - t.lq + 1)); };
    return {upto(last), wlast < r0 ? 0 : upto(wlast), wlast < r0 ? 0 : upto(r0)};
}

// Workgroup id -> (key head, slot, part).  Consecutive ids go round the 8 XCDs, each with an L2 of its own: an XCD gets whole key heads, or every c-th slot of one when the heads
// are not a multiple of 8 -- the tiles that stream one head's rows share an L2, and long and short sequences (causal: early and late tiles) are spread evenly over the XCDs.
struct Work { int head, slot, part; };
__host__ __device__ __forceinline__ int xcd_classes(int heads) { return heads % 8 == 0 ? 1 : heads % 4 == 0 ? 2 : heads % 2 == 0 ? 4 : 8; }
__host__ __device__ __forceinline__ long work_groups(long slots, int heads, int parts) { const int c = xcd_classes(heads); return (slots + c - 1) / c * c * heads * parts; }
__device__ __forceinline__ Work find_work(int id, int heads, int parts) {
    const int c = xcd_classes(heads), units = heads * c / 8;  // (head, slot class) pairs per XCD
    int j = id / 8;
    Work w;
    w.part = j % parts; j /= parts;
    const int unit = id % 8 * units + j % units;
    w.head = unit / c; w.slot = j / units * c + unit % c;
    return w;
}

__device__ __forceinline__ float max_halves(float x) {        // max over lane and lane ^ 32, in both
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// joins the parts of a row: o = sum_s 2^(lse_s - top) o_s / sum_s 2^(lse_s - top); one wave per row, its lanes hold the parts' weights (nsplit <= 64), then D / 64 channels each.
// U parts' reads in flight: latency, 6 us for 8 tokens x 32 heads x 39 parts.
template <typename T, int D, int U>
__global__ void __launch_bounds__(NT) varlen_join_kernel(const VarlenParams<T> p) {
    constexpr int C = D / 64;
    const long rows = p.tq * p.hq, row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= rows) return;
    const int lane = threadIdx.x & 63;
    const long tok = row / p.hq, at = (row - tok * p.hq) * p.tq + tok;
    const float ls = lane < p.nsplit ? p.part_lse[lane * rows + at] : -INFINITY;
    const float top = wave_max(ls), base = top == -INFINITY ? 0.f : top;
    const float w = __builtin_amdgcn_exp2f(ls - base), sum = wave_sum(w);
    float a[C];
#pragma unroll
    for (int c = 0; c < C; ++c) a[c] = 0.f;
    for (int s0 = 0; s0 < p.nsplit; s0 += U) {
        float v[U][C];
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int c = 0; c < C; ++c) v[j][c] = p.part[(min(s0 + j, p.nsplit - 1) * rows + row) * D + lane * C + c];
#pragma unroll
        for (int j = 0; j < U; ++j) {                          // a part that saw nothing has stored nothing: what is read there does not count
            const int s = min(s0 + j, 63);
            const float ws = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s));
            const bool stored = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ls), s)) != -INFINITY;      // (lanes from nsplit on hold -inf)
#pragma unroll
            for (int c = 0; c < C; ++c) a[c] += stored ? ws * v[j][c] : 0.f;
        }
    }
    const float inv = sum > 0.f ? 1.f / sum : sum;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        a[c] *= inv;
        const T hi = Elem<T>::from_f(a[c]);
        p.o[row * D + lane * C + c] = hi;
        if (p.o_lo) p.o_lo[row * D + lane * C + c] = Elem<T>::from_f(a[c] - Elem<T>::to_f(hi));
    }
    if (lane == 0 && p.lse) p.lse[at] = sum == 0.f ? INFINITY : base + __builtin_amdgcn_logf(sum);
}

// sums of parts in order, one thread per 4 channels, one tensor per blockIdx.y; HBM: dK and dV of 9377 keys x 8 heads x 128 in 3 parts in 42 us = 6.5 TB/s
template <typename T>
__global__ void __launch_bounds__(256) varlen_sum_kernel(const float* __restrict__ part, T* first, T* second, int parts, long elements) {
    const long at = 4 * ((long)blockIdx.x * 256 + threadIdx.x);
    if (at >= elements) return;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < parts; ++s) {
        const float4 x = *reinterpret_cast<const float4*>(part + ((long)s * gridDim.y + blockIdx.y) * elements + at);
        a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
    }
    T* out = (blockIdx.y ? second : first) + at;
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
    else *reinterpret_cast<float4*>(out) = a;
}
template <typename T> void sum_parts(const VarlenParams<T>& p, T* first, T* second, int parts, long elements, hipStream_t s) {
    varlen_sum_kernel<T><<<dim3((unsigned)cdiv(elements, 1024), second ? 2 : 1), 256, 0, s>>>(p.part, first, second, parts, elements);
}

inline int row_slots(long tokens, int g, int n, int per) { return (int)(tokens * g / per + n + 1); }

template <typename T, int D> void join(const VarlenParams<T>& p, hipStream_t s) {
    const unsigned grid = (unsigned)cdiv(p.tq * p.hq, 4);
    if (p.nsplit <= 4) varlen_join_kernel<T, D, 4><<<grid, NT, 0, s>>>(p); else varlen_join_kernel<T, D, 16><<<grid, NT, 0, s>>>(p);
}

// attention_varlen_f32.hip
void forward_f32(const VarlenParams<float>& p, int D, hipStream_t s);
void backward_f32(const VarlenParams<float>& p, int D, hipStream_t s);

}  // namespace dpipe_varlen
