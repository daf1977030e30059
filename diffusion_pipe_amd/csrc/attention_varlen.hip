// attention_varlen.hip -- attention over sequences of different lengths packed back to back, with grouped heads, causal or not, forward + backward; bf16.
//
//   q [Tq, Hq, D], k / v [Tk, Hk, D] (head dim contiguous, D in {64, 128}), sequence b = query tokens cu_q[b] .. cu_q[b + 1] and key tokens cu_k[b] .. cu_k[b + 1];
//   query head h reads key head h / g, g = Hq / Hk;  o_i = sum_j softmax_j(scale q_i . k_j) v_j;  causal: key j (counted in its sequence) is seen from query i
//   when j - len_k <= i - len_q.  A query that sees no key gives o = 0 and zero gradients; so do the rows behind the last sequence.
//   lse [Hq][Tq] fp32 in log2 units:  P = exp2(scale log2(e) q . k - lse);  +inf for a query that sees nothing.
//   backward:  delta = rowsum(dO . O);  dV = P^T dO;  dS = P (dO V^T - delta);  dQ = scale dS K;  dK = scale dS^T Q (summed over the g query heads).
//
// Rows: the g query heads that share a key head are one list of len_q * g rows (row r = token r / g, head r % g), so a single token already fills g rows of a tile and the
// shared K / V are staged once for all of them; the dK / dV kernel walks the g heads and sums in registers (no atomics, one fixed order).
// Tiles: sequence b owns the tile slots from  cu[b] * g / TILE + b  on -- at least ceil(rows / TILE) of them for any lengths, at most N + 1 unused ones in all --
// so the grid follows from Tq, N and g alone; a workgroup finds its sequence with one wave-wide comparison, and neither the host nor a planning kernel has to know a length.
// Few rows against long keys: the key range of every sequence is cut into `nsplit` parts (own workgroups, fp32 partial rows) that a second kernel joins.
//
// As in attention.hip everything is v_mfma_f32_32x32x16_bf16 on the transposed score tile S^T = K . Q^T (a lane owns one query column: softmax statistics are
// lane-local), tiles stream global -> LDS by buffer_load ... lds into a two-deep ring of lds_dma_tiles.h images; rows past a sequence's end come back as zeros from the
// buffer bounds check, whatever the neighbouring sequence holds.  Each tile has a buffer descriptor of its own, so a sequence may span more than 4 GiB.
#include <cstdio>
#include "dpipe_common.h"
#include "lds_dma_tiles.h"
#include "attention_tiles.h"
#include "../../include/dpipe_hip.h"

using namespace dpipe;
using namespace dpipe_tiles;

namespace {

struct VarlenParams {
    const bf16_t *q, *k, *v, *dout;
    bf16_t *o, *dq, *dk, *dv;
    float *lse, *delta, *o32;            // lse / delta [Hq][Tq]; o32 [Tq][Hq][D]: the unrounded output, kept for the backward's delta (may be null in the forward)
    const int *cu_q, *cu_k;
    float *part, *part_lse;              // split forms: forward rows [split][Tq][Hq][D] and their lse [split][Hq][Tq]; dK / dV [split][2][Tk][Hk][D]
    long tq, tk;
    int n, hq, hk, g, slots, nsplit, causal;
    long q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, do_ss, do_sh;    // o, dq, dk, dv are contiguous
    float scale;
};

constexpr int KT = 64;                   // keys (dK / dV: queries) per LDS tile
constexpr float M_INIT = -3.0e38f;       // running maximum before the first key: finite, so that exp2(-inf - m) is 0 and never NaN
constexpr float RESCALE_AT = 8.f;        // the accumulator is rescaled when the maximum grew by more than 2^8: P stays below 256, its relative rounding is the same

// ------------------------------------------------------------------------------------------------ which sequence, which rows
struct Tile { int b; long row0, rows; long q0, k0; int lq, lk; bool live; };

__device__ __forceinline__ long bound(const int* cu, int i, int n, long total) {
    if (i == 0) return 0;
    if (i > n) return total;
    const long c = cu[i];
    return c < 0 ? 0 : c > total ? total : c;
}
// slot -> sequence (n: the rows behind the last one) and its first row; PER = rows per tile, gg = rows per token on the tiled side
template <int PER>
__device__ __forceinline__ Tile find_tile(const VarlenParams& p, int slot, bool keys, bool reversed) {
    const int* cu = keys ? p.cu_k : p.cu_q;
    const long total = keys ? p.tk : p.tq;
    const int gg = keys ? 1 : p.g, lane = threadIdx.x & 63;
    int count = 0;
    for (int base = 0; base <= p.n; base += 64) {
        const int i = base + lane;
        const bool at = i <= p.n && bound(cu, i, p.n, total) * gg / PER + i <= slot;
        const int c = __popcll(__ballot(at));
        count += c;
        if (c < 64) break;
    }
    Tile t;
    t.b = __builtin_amdgcn_readfirstlane(count - 1);
    const bool tail = t.b >= p.n;
    const long s0 = bound(cu, t.b, p.n, total), s1 = max(s0, bound(cu, t.b + 1, p.n, total));
    const long rows = (s1 - s0) * gg;
    const int at = slot - (int)(s0 * gg / PER + t.b), nt = (int)((rows + PER - 1) / PER);
    t.live = at >= 0 && at < nt;         // (offsets that do not ascend reach no row outside their tensor)
    t.row0 = (long)(reversed ? nt - 1 - at : at) * PER;
    t.rows = rows;
    long o0 = 0, o1 = 0;                 // the other side of the sequence; the rows behind the last sequence have none
    if (!tail) {
        const int* cu2 = keys ? p.cu_q : p.cu_k;
        const long total2 = keys ? p.tq : p.tk;
        o0 = bound(cu2, t.b, p.n, total2); o1 = max(o0, t.b + 1 > p.n ? o0 : bound(cu2, t.b + 1, p.n, total2));
    }
    t.q0 = keys ? o0 : s0; t.k0 = keys ? s0 : o0;
    t.lq = (int)(keys ? o1 - o0 : s1 - s0); t.lk = (int)(keys ? s1 - s0 : o1 - o0);
    return t;
}

// consecutive workgroup ids go round the 8 XCDs: each XCD gets a contiguous run of (head, slot), so tiles that stream the same K / V share an L2
__device__ __forceinline__ int xcd_order(int id, int total) {
    const int per = total / 8, rest = total % 8, x = id % 8;
    return (x < rest ? x * (per + 1) : rest * (per + 1) + (x - rest) * per) + id / 8;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* base, long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}
// descriptor of up to KT rows of D bf16 (pitch ss) from row `at` on of `n`
template <int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const bf16_t* base, long ss, int at, int n) {
    const int rows = min(n - at, KT);
    return tile_rsrc(base + (long)at * ss, rows > 0 ? ((rows - 1) * ss + D) * 2 : 0);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, char* dst, unsigned off) { __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)dst, 16, off, 0, 0, 0); }
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rs, char* dst, unsigned off) { __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)dst, 4, off, 0, 0, 0); }

template <int D, int NW> struct Offsets {                     // per-lane source offsets of this wave's DMA pieces of one tile
    static constexpr int PP = KT * D * 2 / 1024 / NW;
    unsigned o[PP];
    template <bool MN> __device__ __forceinline__ void init(int wid, int lane, long ss) {
#pragma unroll
        for (int j = 0; j < PP; ++j) {
            const int P = j * NW + wid;
            o[j] = MN ? dma_voffset<true, D>(P, lane, 0, ss) : dma_voffset<false, KT>(P % 8, lane, 0, ss) + (unsigned)(P / 8) * 128u;
        }
    }
    __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t rs, char* img, int wid) const {
#pragma unroll
        for (int j = 0; j < PP; ++j) dma16(rs, img + (j * NW + wid) * 1024, o[j]);
    }
};

__device__ __forceinline__ float max_halves(float x) {        // max over lane and lane ^ 32, in both
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ================================================================================================ forward
template <int D, int QB, int NW, bool SPLIT>
__global__ void __launch_bounds__(NW * 64, (NW == 8 || D == 64) && QB == 1 ? 2 : 1) varlen_fwd_kernel(const VarlenParams p) {
    constexpr int QW = 32 * QB, QWG = QW * NW, NKS = D / 16, NDB = D / 32, IMG = KT * D * 2, STAGE = 2 * IMG;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
    int L = xcd_order(blockIdx.x, gridDim.x);
    const int split = SPLIT ? L % p.nsplit : 0;
    if (SPLIT) L /= p.nsplit;
    const int kh = L / p.slots;
    const Tile t = find_tile<QWG>(p, L % p.slots, false, p.causal);
    if (!t.live) return;

    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const long r0 = t.row0 + wid * QW;                         // first row of this wave
    const int seen = t.lk - t.lq;                              // causal: token x sees keys 0 .. x + seen
    const bf16_t* K = p.k + t.k0 * p.k_ss + kh * p.k_sh;
    const bf16_t* V = p.v + t.k0 * p.v_ss + kh * p.v_sh;
    const float sl2 = p.scale * LOG2E;

    bf16x8_t qf[QB][NKS];
    long orow[QB];                                             // (token * Hq + head) of the lane's rows, -1: none
    int lim[QB];                                               // last key the row sees
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const long r = r0 + 32 * qb + i;
        const bool live = r < t.rows;
        const unsigned tok = live ? (unsigned)r / (unsigned)p.g : 0u, hd = live ? (unsigned)r - tok * (unsigned)p.g : 0u;
        orow[qb] = live ? (t.q0 + tok) * p.hq + kh * p.g + hd : -1;
        lim[qb] = p.causal ? (int)min((long)tok + seen, (long)t.lk - 1) : t.lk - 1;
        const bf16_t* Q = p.q + (t.q0 + tok) * p.q_ss + (long)(kh * p.g + hd) * p.q_sh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) qf[qb][ks] = live ? *reinterpret_cast<const bf16x8_t*>(Q + 16 * ks + 8 * h) : zero_frag();
    }
    f32x16 oacc[QB][NDB];
    float m[QB], l[QB];                                        // m: running maximum in log2 units; l: this lane's part of the sum
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
        for (int db = 0; db < NDB; ++db) oacc[qb][db] = zero16();
        m[qb] = M_INIT; l[qb] = 0.f;
    }

    // keys that any row of the workgroup / every row of the wave sees (wave-uniform)
    const long last = min(t.row0 + QWG, t.rows) - 1, wlast = min(r0 + QW, t.rows) - 1;
    const int wg_keys = p.causal ? (int)max(0l, min((long)t.lk, last / p.g + seen + 1)) : t.lk;
    const int w_keys = wlast < r0 ? 0 : p.causal ? (int)max(0l, min((long)t.lk, wlast / p.g + seen + 1)) : t.lk;
    const int w_full = wlast < r0 ? 0 : p.causal ? (int)max(0l, min((long)t.lk, r0 / p.g + seen + 1)) : t.lk;
    const int nkt = (wg_keys + KT - 1) / KT;
    int kt0 = 0, kt1 = nkt;
    if (SPLIT) {                                               // every part of the sequence's key tiles, cut by its full length
        const int all = (t.lk + KT - 1) / KT, per = (all + p.nsplit - 1) / p.nsplit;
        kt0 = min(nkt, split * per); kt1 = min(nkt, kt0 + per);
    }
    Offsets<D, NW> oK, oV;
    oK.template init<false>(wid, lane, p.k_ss); oV.template init<true>(wid, lane, p.v_ss);
    auto issue = [&](int kt, int buf) {
        char* base = lds + buf * STAGE;
        oK.issue(rows_rsrc<D>(K, p.k_ss, kt * KT, t.lk), base, wid);
        oV.issue(rows_rsrc<D>(V, p.v_ss, kt * KT, t.lk), base + IMG, wid);
    };
    if (kt0 < kt1) issue(kt0, kt0 & 1);
    for (int kt = kt0; kt < kt1; ++kt) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // this wave's pieces of tile kt
        __builtin_amdgcn_s_barrier();                          // everyone's pieces landed; everyone is done with the other buffer
        if (kt + 1 < kt1) issue(kt + 1, (kt + 1) & 1);
        const char* Kl = lds + (kt & 1) * STAGE;
        const char* Vl = Kl + IMG;
        const int key0 = kt * KT;
        if (key0 >= w_keys) continue;                          // wave-uniform: no row of this wave sees the tile
        f32x16 s[QB][2];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) { s[qb][0] = zero16(); s[qb][1] = zero16(); }
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            const bf16x8_t k0f = read_frag<false, KT>(Kl + (ks / 4) * (KT * 128), 0, ks & 3, lane), k1f = read_frag<false, KT>(Kl + (ks / 4) * (KT * 128), 32, ks & 3, lane);
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) { s[qb][0] = mfma16(k0f, qf[qb][ks], s[qb][0]); s[qb][1] = mfma16(k1f, qf[qb][ks], s[qb][1]); }
        }
        bf16x8_t pf[QB][4];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            if (key0 + KT > w_full) {                          // some row of the wave does not see the whole tile
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int key = key0 + 32 * kb + (e & 3) + 8 * (e >> 2) + 4 * h;
                        s[qb][kb][e] = key <= lim[qb] ? s[qb][kb][e] : -INFINITY;
                    }
            }
            float mx = s[qb][0][0];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[qb][kb][e]);
            mx = max_halves(mx) * sl2;
            if (!__all(mx <= m[qb] + RESCALE_AT)) {
                const float m_new = fmaxf(m[qb], mx), alpha = __builtin_amdgcn_exp2f(m[qb] - m_new);
                l[qb] *= alpha; m[qb] = m_new;
#pragma unroll
                for (int db = 0; db < NDB; ++db)
#pragma unroll
                    for (int e = 0; e < 16; ++e) oacc[qb][db][e] *= alpha;
            }
            const float mm = m[qb];
            float rs = 0.f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) { const float pe = __builtin_amdgcn_exp2f(s[qb][kb][e] * sl2 - mm); s[qb][kb][e] = pe; rs += pe; }
            l[qb] += rs;
#pragma unroll
            for (int u = 0; u < 4; ++u) pf[qb][u] = pack_frag(s[qb][u >> 1], 8 * (u & 1));
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)                            // O^T += V^T . P^T
#pragma unroll
            for (int db = 0; db < NDB; ++db) {
                const bf16x8_t vf = read_frag_tr_acc<D>(Vl, 32 * db, 16 * u, lane);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) oacc[qb][db] = mfma16(vf, pf[qb][u], oacc[qb][db]);
            }
    }

#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const float lsum = sum_halves(l[qb]);
        if (orow[qb] < 0) continue;
        const float inv = lsum > 0.f ? 1.f / lsum : (lsum == 0.f ? 0.f : lsum);          // nothing seen: 0;  NaN stays NaN
        const long tok = orow[qb] / p.hq, hd = orow[qb] - tok * p.hq;
        const float lse = lsum == 0.f ? (SPLIT ? -INFINITY : INFINITY) : m[qb] + __builtin_amdgcn_logf(lsum);      // v_log_f32 = log2
        float* f32 = SPLIT ? p.part + ((long)split * p.tq * p.hq + orow[qb]) * D : p.o32 ? p.o32 + orow[qb] * D : nullptr;
        if (h == 0 && (SPLIT || p.lse)) (SPLIT ? p.part_lse + (long)split * p.tq * p.hq : p.lse)[hd * p.tq + tok] = lse;
        if (SPLIT && lsum == 0.f) continue;                    // the join does not read this row
        bf16_t* O = p.o + orow[qb] * D;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int eg = 0; eg < 4; ++eg) {
                const float4 v = make_float4(oacc[qb][db][4 * eg] * inv, oacc[qb][db][4 * eg + 1] * inv, oacc[qb][db][4 * eg + 2] * inv, oacc[qb][db][4 * eg + 3] * inv);
                const int d = 32 * db + 8 * eg + 4 * h;
                if (!SPLIT) *reinterpret_cast<uint2*>(O + d) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
                if (f32) *reinterpret_cast<float4*>(f32 + d) = v;
            }
    }
}

// joins the parts of a row: o = sum_s 2^(lse_s - top) o_s / sum_s 2^(lse_s - top); one thread per 4 channels
template <int D>
__global__ void __launch_bounds__(256) varlen_join_kernel(const VarlenParams p) {
    const long idx = (long)blockIdx.x * 256 + threadIdx.x, rows = p.tq * p.hq, row = idx / (D / 4);
    if (row >= rows) return;
    const int d = 4 * (int)(idx % (D / 4));
    const long tok = row / p.hq, hd = row - tok * p.hq, at = hd * p.tq + tok;
    float top = -INFINITY;
    for (int s = 0; s < p.nsplit; ++s) top = fmaxf(top, p.part_lse[s * rows + at]);
    const float base = top == -INFINITY ? 0.f : top;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int s = 0; s < p.nsplit; ++s) {
        const float ls = p.part_lse[s * rows + at];
        if (ls == -INFINITY) continue;
        const float w = __builtin_amdgcn_exp2f(ls - base);
        const float4 v = *reinterpret_cast<const float4*>(p.part + (s * rows + row) * D + d);
        a.x += w * v.x; a.y += w * v.y; a.z += w * v.z; a.w += w * v.w; sum += w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    a.x *= inv; a.y *= inv; a.z *= inv; a.w *= inv;
    *reinterpret_cast<uint2*>(p.o + row * D + d) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
    if (p.o32) *reinterpret_cast<float4*>(p.o32 + row * D + d) = a;
    if (d == 0 && p.lse) p.lse[at] = sum == 0.f ? INFINITY : base + __builtin_amdgcn_logf(sum);
}

// ================================================================================================ backward: dQ (and delta)
// Per 64-key tile three images: K by rows (S^T = K . Q^T), K transposed (dQ^T += K^T . dS^T), V by rows (dP^T = V . dO^T).
template <int D, int QB, int NW>
__global__ void __launch_bounds__(NW * 64, (NW == 8 || D == 64) && QB == 1 ? 2 : 1) varlen_dq_kernel(const VarlenParams p) {
    constexpr int QW = 32 * QB, QWG = QW * NW, NKS = D / 16, NDB = D / 32, IMG = KT * D * 2, STAGE = 3 * IMG;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
    const int L = xcd_order(blockIdx.x, gridDim.x);
    const int kh = L / p.slots;
    const Tile t = find_tile<QWG>(p, L % p.slots, false, p.causal);
    if (!t.live) return;

    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const long r0 = t.row0 + wid * QW;
    const int seen = t.lk - t.lq;
    const bf16_t* K = p.k + t.k0 * p.k_ss + kh * p.k_sh;
    const bf16_t* V = p.v + t.k0 * p.v_ss + kh * p.v_sh;
    const float sl2 = p.scale * LOG2E;

    bf16x8_t qf[QB][NKS], dof[QB][NKS];
    long orow[QB];
    int lim[QB];
    float lse[QB], dl[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const long r = r0 + 32 * qb + i;
        const bool live = r < t.rows;
        const unsigned tok = live ? (unsigned)r / (unsigned)p.g : 0u, hd = live ? (unsigned)r - tok * (unsigned)p.g : 0u;
        const long head = kh * p.g + hd;
        orow[qb] = live ? (t.q0 + tok) * p.hq + head : -1;
        lim[qb] = p.causal ? (int)min((long)tok + seen, (long)t.lk - 1) : t.lk - 1;
        const bf16_t* Q = p.q + (t.q0 + tok) * p.q_ss + head * p.q_sh;
        const bf16_t* DO = p.dout + (t.q0 + tok) * p.do_ss + head * p.do_sh;
        float d = 0.f;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            qf[qb][ks] = live ? *reinterpret_cast<const bf16x8_t*>(Q + 16 * ks + 8 * h) : zero_frag();
            dof[qb][ks] = live ? *reinterpret_cast<const bf16x8_t*>(DO + 16 * ks + 8 * h) : zero_frag();
            if (live) {
                const float4 a = *reinterpret_cast<const float4*>(p.o32 + orow[qb] * D + 16 * ks + 8 * h), c = *reinterpret_cast<const float4*>(p.o32 + orow[qb] * D + 16 * ks + 8 * h + 4);
                const float of[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) d += of[e] * bf16_to_f32((bf16_t)dof[qb][ks][e]);
            }
        }
        dl[qb] = sum_halves(d);
        const long at = head * p.tq + t.q0 + tok;
        lse[qb] = live ? p.lse[at] : INFINITY;
        if (live && h == 0) p.delta[at] = dl[qb];
    }
    f32x16 dq[QB][NDB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int db = 0; db < NDB; ++db) dq[qb][db] = zero16();

    const long last = min(t.row0 + QWG, t.rows) - 1, wlast = min(r0 + QW, t.rows) - 1;
    const int wg_keys = p.causal ? (int)max(0l, min((long)t.lk, last / p.g + seen + 1)) : t.lk;
    const int w_keys = wlast < r0 ? 0 : p.causal ? (int)max(0l, min((long)t.lk, wlast / p.g + seen + 1)) : t.lk;
    const int w_full = wlast < r0 ? 0 : p.causal ? (int)max(0l, min((long)t.lk, r0 / p.g + seen + 1)) : t.lk;
    const int nkt = (wg_keys + KT - 1) / KT;

    Offsets<D, NW> oKc, oKm, oVc;
    oKc.template init<false>(wid, lane, p.k_ss); oKm.template init<true>(wid, lane, p.k_ss); oVc.template init<false>(wid, lane, p.v_ss);
    auto issue = [&](int kt) {
        char* base = lds + (kt & 1) * STAGE;
        const auto rk = rows_rsrc<D>(K, p.k_ss, kt * KT, t.lk);
        oKc.issue(rk, base, wid); oKm.issue(rk, base + IMG, wid);
        oVc.issue(rows_rsrc<D>(V, p.v_ss, kt * KT, t.lk), base + 2 * IMG, wid);
    };
    if (nkt > 0) issue(0);
    for (int kt = 0; kt < nkt; ++kt) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (kt + 1 < nkt) issue(kt + 1);
        const char* Kc = lds + (kt & 1) * STAGE;
        const char* Km = Kc + IMG;
        const char* Vc = Kc + 2 * IMG;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int key0 = kt * KT + 32 * kb;
            if (key0 >= w_keys) break;
            f32x16 s[QB], dp[QB];
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) { s[qb] = zero16(); dp[qb] = zero16(); }
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                const bf16x8_t kf = read_frag<false, KT>(Kc + (ks / 4) * (KT * 128), 32 * kb, ks & 3, lane), vf = read_frag<false, KT>(Vc + (ks / 4) * (KT * 128), 32 * kb, ks & 3, lane);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) { s[qb] = mfma16(kf, qf[qb][ks], s[qb]); dp[qb] = mfma16(vf, dof[qb][ks], dp[qb]); }
            }
            bf16x8_t ds[QB][2];
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                if (key0 + 32 > w_full) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[qb][e] = key0 + (e & 3) + 8 * (e >> 2) + 4 * h <= lim[qb] ? s[qb][e] : -INFINITY;
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) s[qb][e] = __builtin_amdgcn_exp2f(s[qb][e] * sl2 - lse[qb]) * (dp[qb][e] - dl[qb]);
                ds[qb][0] = pack_frag(s[qb], 0); ds[qb][1] = pack_frag(s[qb], 8);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int db = 0; db < NDB; ++db) {
                    const bf16x8_t kf = read_frag_tr_acc<D>(Km, 32 * db, 32 * kb + 16 * u, lane);
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb) dq[qb][db] = mfma16(kf, ds[qb][u], dq[qb][db]);
                }
        }
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        if (orow[qb] < 0) continue;
        bf16_t* DQ = p.dq + orow[qb] * D;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int eg = 0; eg < 4; ++eg)
                *reinterpret_cast<uint2*>(DQ + 32 * db + 8 * eg + 4 * h) =
                    make_uint2(pack_bf16x2(dq[qb][db][4 * eg] * p.scale, dq[qb][db][4 * eg + 1] * p.scale), pack_bf16x2(dq[qb][db][4 * eg + 2] * p.scale, dq[qb][db][4 * eg + 3] * p.scale));
    }
}

// ================================================================================================ backward: dK, dV
// Key-outer; a lane owns one key column per block:  S = Q . K^T, dP = dO . V^T, dV^T += dO^T . P, dK^T += Q^T . dS.  Per 64-query tile four images (Q and dO, by rows and
// transposed) and the tile's lse / delta.  Query rows past the sequence arrive as zeros (Q, dO, lse, delta): P = 1 there, but dO = 0 and dS = 0.  MODE 0: both; 1: dV; 2: dK.
template <int D, int KB, int NW, int MODE>
__global__ void __launch_bounds__(NW * 64, (NW == 8 || D == 64) && KB == 1 ? 2 : 1) varlen_dkv_kernel(const VarlenParams p) {
    constexpr bool DO_K = MODE != 1, DO_V = MODE != 2;
    constexpr int KW = 32 * KB, KWG = KW * NW, QT = 64, NKS = D / 16, NDB = D / 32, IMG = QT * D * 2, NIMG = 1 + (DO_V ? 1 : 0) + (DO_K ? 2 : 0), STAGE = NIMG * IMG + 1024;
    constexpr int O_DOM = IMG, O_DOC = (1 + (DO_V ? 1 : 0)) * IMG, O_QM = O_DOC + IMG, O_STAT = NIMG * IMG;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
    int L = xcd_order(blockIdx.x, gridDim.x);
    const int split = L % p.nsplit;
    L /= p.nsplit;
    const int kh = L / p.slots;
    const Tile t = find_tile<KWG>(p, L % p.slots, true, false);
    if (!t.live) return;

    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const int k0w = (int)t.row0 + wid * KW;                    // first key of this wave
    const int seen = t.lk - t.lq;
    const float sl2 = p.scale * LOG2E;
    bf16x8_t kf[KB][NKS], vf[KB][NKS];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int key = k0w + 32 * kb + i;
        const bool live = key < t.lk;
        const bf16_t* K = p.k + (t.k0 + (live ? key : 0)) * p.k_ss + kh * p.k_sh;
        const bf16_t* V = p.v + (t.k0 + (live ? key : 0)) * p.v_ss + kh * p.v_sh;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) {
            kf[kb][ks] = live ? *reinterpret_cast<const bf16x8_t*>(K + 16 * ks + 8 * h) : zero_frag();
            if constexpr (DO_K) vf[kb][ks] = live ? *reinterpret_cast<const bf16x8_t*>(V + 16 * ks + 8 * h) : zero_frag();
        }
    }
    f32x16 dk[KB][NDB], dv[KB][NDB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int db = 0; db < NDB; ++db) { dk[kb][db] = zero16(); dv[kb][db] = zero16(); }

    // query tiles: from the first one that sees a key of this workgroup, for each of the g heads
    const int qt0 = p.causal ? max(0, (int)t.row0 - seen) / QT : 0;
    const int per_head = max(0, (t.lq + QT - 1) / QT - qt0);
    const long all = (long)per_head * p.g, per = (all + p.nsplit - 1) / p.nsplit;
    const int it0 = (int)min(all, split * per), it1 = (int)min(all, it0 + per);

    Offsets<D, NW> oQc, oQm, oDc, oDm;
    oQc.template init<false>(wid, lane, p.q_ss); oQm.template init<true>(wid, lane, p.q_ss);
    oDc.template init<false>(wid, lane, p.do_ss); oDm.template init<true>(wid, lane, p.do_ss);
    auto issue = [&](int it, int buf) {
        const int hd = it / per_head, q = (qt0 + it - hd * per_head) * QT;
        const long head = kh * p.g + hd;
        char* base = lds + buf * STAGE;
        const auto rq = rows_rsrc<D>(p.q + t.q0 * p.q_ss + head * p.q_sh, p.q_ss, q, t.lq), rd = rows_rsrc<D>(p.dout + t.q0 * p.do_ss + head * p.do_sh, p.do_ss, q, t.lq);
        oQc.issue(rq, base, wid);
        if constexpr (DO_V) oDm.issue(rd, base + O_DOM, wid);
        if constexpr (DO_K) { oDc.issue(rd, base + O_DOC, wid); oQm.issue(rq, base + O_QM, wid); }
        const int rows = min(QT, t.lq - q);
        if (wid == 0) dma4(tile_rsrc(p.lse + head * p.tq + t.q0 + q, rows * 4), base + O_STAT, lane * 4);
        if (DO_K && wid == 1) dma4(tile_rsrc(p.delta + head * p.tq + t.q0 + q, rows * 4), base + O_STAT + 256, lane * 4);
    };
    if (it0 < it1) issue(it0, 0);
    for (int it = it0; it < it1; ++it) {
        const int buf = (it - it0) & 1;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (it + 1 < it1) issue(it + 1, buf ^ 1);
        const int q00 = (qt0 + it % per_head) * QT;
        const char* Qc = lds + buf * STAGE;
        const char* DOm = Qc + O_DOM;
        const char* DOc = Qc + O_DOC;
        const char* Qm = Qc + O_QM;
        const float* lse_l = reinterpret_cast<const float*>(Qc + O_STAT);
        const float* dl_l = lse_l + 64;
        if (k0w >= t.lk) continue;                             // wave-uniform: no live key
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
            const int q0 = q00 + 32 * qb;
            if (q0 >= t.lq) break;
            if (p.causal && q0 + 31 + seen < k0w) continue;    // no query of the block sees a key of this wave
            f32x16 s[KB], dp[KB];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) { s[kb] = zero16(); dp[kb] = zero16(); }
#pragma unroll
            for (int ks = 0; ks < NKS; ++ks) {
                const bf16x8_t qf = read_frag<false, QT>(Qc + (ks / 4) * (QT * 128), 32 * qb, ks & 3, lane);
#pragma unroll
                for (int kb = 0; kb < KB; ++kb) s[kb] = mfma16(qf, kf[kb][ks], s[kb]);
                if constexpr (DO_K) {
                    const bf16x8_t df = read_frag<false, QT>(DOc + (ks / 4) * (QT * 128), 32 * qb, ks & 3, lane);
#pragma unroll
                    for (int kb = 0; kb < KB; ++kb) dp[kb] = mfma16(df, vf[kb][ks], dp[kb]);
                }
            }
            const bool masked = p.causal && q0 + seen < k0w + KW - 1;      // some query of the block does not see every key of this wave
            bf16x8_t pf[KB][2], ds[KB][2];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const int key = k0w + 32 * kb + i;
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[kb][e] = key <= q0 + 8 * (e >> 2) + 4 * h + (e & 3) + seen ? s[kb][e] : -INFINITY;
                }
                f32x16 pr;
#pragma unroll
                for (int eg = 0; eg < 4; ++eg) {
                    const float4 l4 = *reinterpret_cast<const float4*>(&lse_l[32 * qb + 8 * eg + 4 * h]);
                    float4 d4 = make_float4(0.f, 0.f, 0.f, 0.f);
                    if constexpr (DO_K) d4 = *reinterpret_cast<const float4*>(&dl_l[32 * qb + 8 * eg + 4 * h]);
                    const float ll[4] = {l4.x, l4.y, l4.z, l4.w}, dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int e = 4 * eg + j;
                        pr[e] = __builtin_amdgcn_exp2f(s[kb][e] * sl2 - ll[j]);
                        s[kb][e] = pr[e] * (dp[kb][e] - dd[j]);
                    }
                }
                pf[kb][0] = pack_frag(pr, 0); pf[kb][1] = pack_frag(pr, 8);
                ds[kb][0] = pack_frag(s[kb], 0); ds[kb][1] = pack_frag(s[kb], 8);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int db = 0; db < NDB; ++db) {
                    if constexpr (DO_V) {
                        const bf16x8_t df = read_frag_tr_acc<D>(DOm, 32 * db, 32 * qb + 16 * u, lane);
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb) dv[kb][db] = mfma16(df, pf[kb][u], dv[kb][db]);
                    }
                    if constexpr (DO_K) {
                        const bf16x8_t qf = read_frag_tr_acc<D>(Qm, 32 * db, 32 * qb + 16 * u, lane);
#pragma unroll
                        for (int kb = 0; kb < KB; ++kb) dk[kb][db] = mfma16(qf, ds[kb][u], dk[kb][db]);
                    }
                }
        }
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        const int key = k0w + 32 * kb + i;
        if (key >= t.lk) continue;
        const long row = ((t.k0 + key) * p.hk + kh) * D, slice = p.tk * p.hk * D;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
            for (int eg = 0; eg < 4; ++eg) {
                const long at = row + 32 * db + 8 * eg + 4 * h;
                const float4 a = make_float4(dk[kb][db][4 * eg] * p.scale, dk[kb][db][4 * eg + 1] * p.scale, dk[kb][db][4 * eg + 2] * p.scale, dk[kb][db][4 * eg + 3] * p.scale);
                const float4 c = make_float4(dv[kb][db][4 * eg], dv[kb][db][4 * eg + 1], dv[kb][db][4 * eg + 2], dv[kb][db][4 * eg + 3]);
                if (p.nsplit > 1) {
                    if constexpr (DO_K) *reinterpret_cast<float4*>(p.part + 2 * split * slice + at) = a;
                    if constexpr (DO_V) *reinterpret_cast<float4*>(p.part + (2 * split + 1) * slice + at) = c;
                } else {
                    if constexpr (DO_K) *reinterpret_cast<uint2*>(p.dk + at) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
                    if constexpr (DO_V) *reinterpret_cast<uint2*>(p.dv + at) = make_uint2(pack_bf16x2(c.x, c.y), pack_bf16x2(c.z, c.w));
                }
            }
    }
}

// dK / dV = sum of the parts in order, one thread per 4 channels
__global__ void __launch_bounds__(256) varlen_dkv_sum_kernel(const VarlenParams p, long elements) {
    const long at = 4 * ((long)blockIdx.x * 256 + threadIdx.x);
    if (at >= elements) return;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), c = a;
#pragma unroll 4
    for (int s = 0; s < p.nsplit; ++s) {
        const float4 x = *reinterpret_cast<const float4*>(p.part + 2 * s * elements + at), y = *reinterpret_cast<const float4*>(p.part + (2 * s + 1) * elements + at);
        a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w; c.x += y.x; c.y += y.y; c.z += y.z; c.w += y.w;
    }
    *reinterpret_cast<uint2*>(p.dk + at) = make_uint2(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w));
    *reinterpret_cast<uint2*>(p.dv + at) = make_uint2(pack_bf16x2(c.x, c.y), pack_bf16x2(c.z, c.w));
}

// ------------------------------------------------------------------------------------------------ host side
int row_slots(long tokens, int g, int n, int per) { return (int)(tokens * g / per + n + 1); }

// parts of the key range: when the row tiles alone leave CUs idle, enough parts for two workgroups per CU, of at least 4 key tiles of an average sequence each
int fwd_splits(long tq, long tk, int n, int hq, int hk) {
    const long wgs = cdiv(tq * (hq / hk), 128) * hk, tiles = tk / n / KT;
    if (wgs >= 256 || tiles < 8) return 1;
    long s = cdiv(512, wgs);
    if (s > tiles / 4) s = tiles / 4;
    return (int)(s > 128 ? 128 : s);
}
// parts of the query range for dK / dV, likewise
int dkv_splits(long tq, long tk, int n, int hq, int hk) {
    const long wgs = cdiv(tk, 128) * hk, tiles = tq / n / 64 * (hq / hk);
    if (wgs >= 256 || tiles < 8) return 1;
    long s = cdiv(512, wgs);
    if (s > tiles / 4) s = tiles / 4;
    return (int)(s > 64 ? 64 : s);
}

bool rows_ok(const void* p, long ss, long sh, int D) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ss % 8 == 0 && sh % 8 == 0 && ss >= D && ss < (1l << 23) && sh >= 0;
}

int fill(VarlenParams& p, const char* what, const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, long tq, long tk, int n, int hq, int hk, int D, long q_ss,
         long q_sh, long k_ss, long k_sh, long v_ss, long v_sh, float scale, int causal) {
    auto bad = [&](const char* m, int rc = DPIPE_ERR_ARG) { char buf[160]; snprintf(buf, sizeof(buf), "%s: %s", what, m); set_last_error(buf); return rc; };
    if (!q || !k || !v || !cu_q || !cu_k || tq <= 0 || tk <= 0 || n <= 0 || hq <= 0 || hk <= 0 || hq % hk) return bad("bad argument");
    if (D != 64 && D != 128) return bad("head dim must be 64 or 128", DPIPE_ERR_UNSUPPORTED);
    if (!(scale > 0.f) || scale > 1e30f) return bad("scale must be positive and finite");
    if (tq * (hq / hk) >= (1l << 31) || tk >= (1l << 31) || ((tq * hq + tk * hk) / 128 + (n + 1l) * hk) * fwd_splits(tq, tk, n, hq, hk) >= (1l << 23) ||
        (tk * hk / 128 + (n + 1l) * hk) * dkv_splits(tq, tk, n, hq, hk) >= (1l << 23)) return bad("too many rows or sequences", DPIPE_ERR_UNSUPPORTED);
    if (!rows_ok(q, q_ss, q_sh, D) || !rows_ok(k, k_ss, k_sh, D) || !rows_ok(v, v_ss, v_sh, D)) return bad("tensors must be 16-byte aligned with strides multiple of 8 elements");
    p.q = (const bf16_t*)q; p.k = (const bf16_t*)k; p.v = (const bf16_t*)v; p.cu_q = cu_q; p.cu_k = cu_k; p.tq = tq; p.tk = tk; p.n = n; p.hq = hq; p.hk = hk; p.g = hq / hk;
    p.q_ss = q_ss; p.q_sh = q_sh; p.k_ss = k_ss; p.k_sh = k_sh; p.v_ss = v_ss; p.v_sh = v_sh; p.scale = scale; p.causal = causal != 0; p.nsplit = 1;
    return DPIPE_OK;
}

template <int D, int QB, int NW, bool SPLIT> void launch_fwd(VarlenParams& p, hipStream_t s) {
    p.slots = row_slots(p.tq, p.g, p.n, 32 * QB * NW);
    varlen_fwd_kernel<D, QB, NW, SPLIT><<<(unsigned)((long)p.slots * p.hk * p.nsplit), NW * 64, 0, s>>>(p);
}
template <int D> void forward(VarlenParams& p, hipStream_t s) {
    if (p.nsplit > 1) {
        launch_fwd<D, 1, 4, true>(p, s);
        varlen_join_kernel<D><<<(unsigned)cdiv(p.tq * p.hq * (D / 4), 256), 256, 0, s>>>(p);
    } else if (cdiv(p.tq * p.g, 256) * p.hk >= 192) {
        launch_fwd<D, 1, 8, false>(p, s);
    } else {
        launch_fwd<D, 1, 4, false>(p, s);
    }
}
template <int D, int QB, int NW> void launch_dq(VarlenParams& p, hipStream_t s) {
    p.slots = row_slots(p.tq, p.g, p.n, 32 * QB * NW);
    varlen_dq_kernel<D, QB, NW><<<(unsigned)((long)p.slots * p.hk), NW * 64, 0, s>>>(p);
}
template <int D, int KB, int NW, int MODE> void launch_dkv(VarlenParams& p, hipStream_t s) {
    p.slots = row_slots(p.tk, 1, p.n, 32 * KB * NW);
    varlen_dkv_kernel<D, KB, NW, MODE><<<(unsigned)((long)p.slots * p.hk * p.nsplit), NW * 64, 0, s>>>(p);
}
template <int D> void backward(VarlenParams& p, int splits, hipStream_t s) {
    if (cdiv(p.tq * p.g, 256) * p.hk >= 192) launch_dq<D, 1, 8>(p, s); else launch_dq<D, 1, 4>(p, s);
    p.nsplit = splits;
    if (D == 128 && splits == 1 && cdiv(p.tk, 256) * p.hk >= 192) { launch_dkv<D, 1, 8, 1>(p, s); launch_dkv<D, 1, 8, 2>(p, s); }
    else launch_dkv<D, 1, 4, 0>(p, s);
    if (splits > 1) { const long e = p.tk * p.hk * D; varlen_dkv_sum_kernel<<<(unsigned)cdiv(e, 1024), 256, 0, s>>>(p, e); }
}

}  // namespace

extern "C" {

long dpipe_attn_varlen_fwd_workspace_floats(long tq, long tk, int n, int hq, int hk, int D) {
    if (tq <= 0 || tk <= 0 || n <= 0 || hq <= 0 || hk <= 0 || hq % hk) return 0;
    const int s = fwd_splits(tq, tk, n, hq, hk);
    return s > 1 ? (long)s * tq * hq * (D + 1) : 0;
}
long dpipe_attn_varlen_bwd_workspace_floats(long tq, long tk, int n, int hq, int hk, int D) {
    if (tq <= 0 || tk <= 0 || n <= 0 || hq <= 0 || hk <= 0 || hq % hk) return 0;
    const int s = dkv_splits(tq, tk, n, hq, hk);
    return s > 1 ? 2l * s * tk * hk * D : 0;
}

int dpipe_attn_varlen_fwd(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, void* o, float* lse, float* o_f32, float* ws, long ws_floats, long tq,
                          long tk, int n, int hq, int hk, int D, long q_ss, long q_sh, long k_ss, long k_sh, long v_ss, long v_sh, float scale, int causal, void* stream) {
    VarlenParams p = {};
    const int rc = fill(p, "dpipe_attn_varlen_fwd", q, k, v, cu_q, cu_k, tq, tk, n, hq, hk, D, q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, scale, causal);
    if (rc) return rc;
    const long need = dpipe_attn_varlen_fwd_workspace_floats(tq, tk, n, hq, hk, D);
    if (!o || !aligned16(o) || !aligned16(o_f32) || (need > 0 && (!ws || ws_floats < need || !aligned16(ws)))) {
        set_last_error("dpipe_attn_varlen_fwd: bad output or workspace"); return DPIPE_ERR_ARG; }
    if (ablated(ABL_ATTN)) return DPIPE_OK;
    p.o = (bf16_t*)o; p.lse = lse; p.o32 = o_f32;
    if (need > 0) { p.nsplit = fwd_splits(tq, tk, n, hq, hk); p.part = ws; p.part_lse = ws + (long)p.nsplit * tq * hq * D; }
    if (D == 64) forward<64>(p, reinterpret_cast<hipStream_t>(stream)); else forward<128>(p, reinterpret_cast<hipStream_t>(stream));
    return check_launch("dpipe_attn_varlen_fwd");
}

int dpipe_attn_varlen_bwd(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, const float* o_f32, const void* dout, const float* lse, float* delta,
                          void* dq, void* dk, void* dv, float* ws, long ws_floats, long tq, long tk, int n, int hq, int hk, int D, long q_ss, long q_sh, long k_ss, long k_sh,
                          long v_ss, long v_sh, long do_ss, long do_sh, float scale, int causal, void* stream) {
    VarlenParams p = {};
    const int rc = fill(p, "dpipe_attn_varlen_bwd", q, k, v, cu_q, cu_k, tq, tk, n, hq, hk, D, q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, scale, causal);
    if (rc) return rc;
    const long need = dpipe_attn_varlen_bwd_workspace_floats(tq, tk, n, hq, hk, D);
    if (!o_f32 || !dout || !lse || !delta || !dq || !dk || !dv || !aligned16(o_f32) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) || !rows_ok(dout, do_ss, do_sh, D) ||
        (need > 0 && (!ws || ws_floats < need || !aligned16(ws)))) { set_last_error("dpipe_attn_varlen_bwd: bad gradient or workspace"); return DPIPE_ERR_ARG; }
    if (ablated(ABL_ATTN)) return DPIPE_OK;
    p.o32 = const_cast<float*>(o_f32); p.dout = (const bf16_t*)dout; p.lse = const_cast<float*>(lse); p.delta = delta;
    p.dq = (bf16_t*)dq; p.dk = (bf16_t*)dk; p.dv = (bf16_t*)dv; p.do_ss = do_ss; p.do_sh = do_sh; p.part = ws;
    const int splits = need > 0 ? dkv_splits(tq, tk, n, hq, hk) : 1;
    if (D == 64) backward<64>(p, splits, reinterpret_cast<hipStream_t>(stream)); else backward<128>(p, splits, reinterpret_cast<hipStream_t>(stream));
    return check_launch("dpipe_attn_varlen_bwd");
}

}  // extern "C"
