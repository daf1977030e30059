// attention_varlen.hip -- attention over sequences of different lengths packed back to back, with grouped heads, causal or not, forward + backward; bf16 (fp32:
// attention_varlen_f32.hip, the same contract).
//
//   q [Tq, Hq, D], k / v [Tk, Hk, D] (head dim contiguous, D in {64, 128}), sequence b = query tokens cu_q[b] .. cu_q[b + 1] and key tokens cu_k[b] .. cu_k[b + 1];
//   query head h reads key head h / g, g = Hq / Hk;  o_i = sum_j softmax_j(scale q_i . k_j) v_j;  causal: key j (counted in its sequence) is seen from query i
//   when j - len_k <= i - len_q.  A query that sees no key gives o = 0 and zero gradients; so do the rows behind the last sequence.
//   lse [Hq][Tq] fp32 in log2 units:  P = exp2(scale log2(e) q . k - lse);  +inf for a query that sees nothing.
//   backward:  delta = rowsum(dO . O);  dV = P^T dO;  dS = P (dO V^T - delta);  dQ = scale dS K;  dK = scale dS^T Q (summed over the g query heads).
//
// Rows: the g query heads that share a key head are one list of len_q * g rows (row r = token r / g, head r % g), so a single token already fills g rows of a tile and the
// shared K / V are staged once for all of them; the dK / dV kernel walks the g heads and sums in registers (no atomics, one fixed order).
// Tiles: there are at most rows / TILE + N + 1 tile slots for any lengths, so the grid follows from Tq, N and g alone; a workgroup finds its sequence in the offsets by itself
// (find_tile), and neither the host nor a planning kernel has to know a length.
// Few rows against long keys: the key range of every sequence is cut into `nsplit` parts (own workgroups, fp32 partial rows) that a second kernel joins.
//
// As in attention.hip everything is v_mfma_f32_32x32x16_bf16 on the transposed score tile S^T = K . Q^T (a lane owns one query column: softmax statistics are
// lane-local), tiles stream global -> LDS by buffer_load ... lds into a two-deep ring; rows past a sequence's end come back as zeros from the
// buffer bounds check, whatever the neighbouring sequence holds.  Each tile has a buffer descriptor of its own, so a sequence may span more than 4 GiB.
//
// Bound: the matrix pipe, and with it the clock -- on long sequences the pipe is 57 - 68 % busy at 1.7 - 1.9 GHz (2.2 where it is less busy), as in a library product of 8192^3
// (70 % at 1.9 GHz, 1238 TFLOP/s).  TFLOP/s of the products each kernel makes (forward 2, dQ 3, dK / dV 4):
//   15000 + 6001 tokens, 24 heads of 128         forward 2.93 ms = 1093    dQ 3.95 ms = 1218    dK / dV 5.53 ms = 1159
//   4608 + 2560 + 1311 tokens, 24 heads of 128            363 us =  999           475 us = 1145             662 us = 1095
//   7 causal sequences, 9277 tokens, 32 / 8 heads of 128  242 us =  831           308 us =  979             446 us =  901
//   4096 + 2501 + 1024 tokens, 10 heads of 64              89 us =  694           107 us =  865             148 us =  832
// The formulas have seven products, these kernels nine: both backward kernels make S and dP, so that dQ needs neither atomics nor a sum over fp32 parts (at 256 keys a part, len_k / 256
// times the bytes of an fp32 dQ, written and read).
#include <cstdio>
#include "dpipe_common.h"
#include "lds_dma_tiles.h"
#include "attention_tiles.h"
#include "attention_varlen.h"
#include "../../include/dpipe_hip.h"

using namespace dpipe;
using namespace dpipe_tiles;
using namespace dpipe_varlen;

namespace {

typedef VarlenParams<bf16_t> Params;

constexpr int KT = 64;                   // keys (dK / dV: queries) per LDS tile
constexpr int AQ = 4, AK = 1;            // steps of LDS operands read ahead of their products in the dQ and the dK / dV kernels
// CORNER: in a row of few keys (a column of few queries) nothing averages the rounding of P and dS away, and the forward's reaches the row's dS through delta.  The forward and dQ
// therefore multiply what the rounding of a sequence's first tile of keys left as well: one tile in lk / 64 (long sequences: within 1 %), and the rows that only see that tile, which
// in causal sequences carry the largest gradients, are rounded once.  dK / dV do it for sequences of one tile of keys and one of queries (those that see keys), whatever else is in
// the batch: they walk their tiles twice, the second time with what the rounding left (64 sequences of 64 tokens, 24 heads of 128, forward and backward: 127 -> 133 us against a kernel
// for batches of short sequences only; longer sequences as without it.  The second products behind the first in the same pass cost the long ones 8 % in registers, at D = 64 30 %; a
// second body for short sequences in the kernel 2 %; the second walk inside a tile's iteration 4 %).  Error against 64 bits, dQ / dK / dV, 24 causal sequences of 1 - 2 tokens:
// 2.53e-3 / 2.32e-3 / 1.82e-3 -> 1.7e-3 each (one rounding); 457 + 16 + 32 + 172 + 208 causal tokens: dQ 2.40e-3 -> 1.8e-3.

__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rsrc(const void* base, long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, (int)bytes, 0x00020000);
}
// descriptor of up to KR rows of D bf16 (pitch ss) from row `at` on of `n`
template <int D, int KR = KT>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const bf16_t* base, long ss, int at, int n) {
    const int rows = min(n - at, KR);
    return tile_rsrc(base + (long)at * ss, rows > 0 ? ((rows - 1) * ss + D) * 2 : 0);
}
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, char* dst, unsigned off) { __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)dst, 16, off, 0, 0, 0); }
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rs, char* dst, unsigned off) { __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)dst, 4, off, 0, 0, 0); }

// LDS image of a tile of KR rows (64 or 32), read both by rows and transposed: slices of 64 columns, [KR rows][128 B] each, 16-byte chunk c of row r at chunk c ^ f(r) with
// f(r) = (r1 r3 r2) in bits of r.  Rows 0 .. 15 of one chunk (ds_read_b128) then cover the 256 B of all banks once, and so do the 4 rows x 64 B of one transposed read's half wave
// (rows r .. r + 3 differ in r0 -- the 128-byte half -- and r1 -- the 64-byte granule).  One image where a tile is needed both ways (K in dQ; Q and dO in dK / dV) halves its DMA
// traffic and its LDS.
__device__ __forceinline__ int swizzle(int r) { return ((r >> 1) & 1) << 2 | ((r >> 2) & 3); }

template <int D, int NW, int KR = KT> struct Offsets {                     // per-lane source offsets of this wave's 1 KiB DMA pieces (8 rows of a slice) of one tile
    static constexpr int PP = KR * D * 2 / 1024 / NW, BLOCKS = KR / 8;
    unsigned o[PP];
    __device__ __forceinline__ void init(int wid, int lane, long ss) {
#pragma unroll
        for (int j = 0; j < PP; ++j) {
            const int P = j * NW + wid, row = 8 * (P % BLOCKS) + (lane >> 3);
            o[j] = (unsigned)(row * ss * 2) + (unsigned)(P / BLOCKS) * 128u + (unsigned)(((lane & 7) ^ swizzle(row)) << 4);
        }
    }
    __device__ __forceinline__ void issue(__amdgpu_buffer_rsrc_t rs, char* img, int wid) const {
#pragma unroll
        for (int j = 0; j < PP; ++j) dma16(rs, img + (j * NW + wid) * 1024, o[j]);
    }
};

// MFMA operand with k along the row: lane (i, h) gets columns 16 ks + 8 h .. + 8 of row `row + i` (row a multiple of 32)
template <int KR = KT> __device__ __forceinline__ bf16x8_t by_rows(const char* img, int row, int ks, int lane) {
    const int i = lane & 31;
    return *reinterpret_cast<const bf16x8_t*>(img + (ks / 4) * (KR * 128) + row * 128 + i * 128 + ((((lane >> 5) ^ swizzle(i)) ^ (2 * (ks & 3))) << 4));
}
// MFMA operand of the transposed tile: m = column `col + i` (col a multiple of 32), k = the rows of the 16-row block r0 in the order a lane holds them in a score accumulator
// ({4 h + 0 .. 3, 8 + 4 h + 0 .. 3}), so P / dS go from their accumulators straight into the product
template <int KR = KT> __device__ __forceinline__ bf16x8_t by_cols(const char* img, int col, int r0, int lane) {
    const int t = lane & 15, g = lane >> 4, r = 4 * (g >> 1) + (t >> 2);
    const char* p = img + (col / 64) * (KR * 128) + r0 * 128 + r * 128 + (t & 1) * 8;
    const int c = (((col / 32) & 1) << 2 | (g & 1) << 1 | ((t & 3) >> 1)) ^ swizzle(r);
    const bf16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_bf16x4_t*)(p + (c << 4)));
    const bf16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_bf16x4_t*)(p + 8 * 128 + ((c ^ 2) << 4)));
    bf16x8_t out;
    out[0] = lo[0]; out[1] = lo[1]; out[2] = lo[2]; out[3] = lo[3];
    out[4] = hi[0]; out[5] = hi[1]; out[6] = hi[2]; out[7] = hi[3];
    return out;
}

// N steps of products whose LDS operands are read AHEAD steps before their use: step j's products, then the reads of step j + AHEAD, in exactly this order.  (Left to itself the
// compiler reads every operand right before its product and waits the LDS latency out each time: 56 % of all wave cycles of the dK / dV kernel.)
template <int AHEAD, typename Frag, typename Load>
__device__ __forceinline__ void ahead_start(Frag (&f)[AHEAD], Load load) {
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) f[j] = load(j);
    __builtin_amdgcn_sched_barrier(0);
}
template <int N, int AHEAD, typename Frag, typename Load, typename Use>
__device__ __forceinline__ void ahead_run(Frag (&f)[AHEAD], Load load, Use use) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        use(j, f[j % AHEAD]);
        if (j + AHEAD < N) f[j % AHEAD] = load(j + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Head size 64: a wave at its products goes before the others of its SIMD, whose exponentials fill the gaps (3 images, 10 heads: forward 96.6 -> 93.5 us, dK / dV 164 -> 158, dQ 1 %;
// at 128, where the clock gives way as the matrix pipe fills, nothing is gained, in dK / dV 3 % lost, and where few rows read long keys 1 %)
template <int D> __device__ __forceinline__ void products_first(bool on) {
    if (D == 64) { if (on) __builtin_amdgcn_s_setprio(1); else __builtin_amdgcn_s_setprio(0); }
}

// what pack_frag's rounding leaves of 8 accumulator entries, itself as an operand
__device__ __forceinline__ bf16x8_t pack_rest(const f32x16& s, int e0) {
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = s[e0 + 2 * i], y = s[e0 + 2 * i + 1];
        const uint32_t w = pack_bf16x2(x, y);
        r[i] = pack_bf16x2(x - __uint_as_float(w << 16), y - __uint_as_float(w & 0xffff0000u));
    }
    return __builtin_bit_cast(bf16x8_t, make_uint4(r[0], r[1], r[2], r[3]));
}

// the same in place, for a whole tile
__device__ __forceinline__ void rounding_left(f32x16& s) {
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
        const uint32_t w = pack_bf16x2(s[e], s[e + 1]);
        s[e] -= __uint_as_float(w << 16); s[e + 1] -= __uint_as_float(w & 0xffff0000u);
    }
}

// 32 channels of a lane's row from a transposed accumulator (the lane holds channels 8 e + 4 h + 0 .. 3): halves exchanged with lane ^ 32, two 16-byte stores a lane.
// `lo`: where the rounding's remainders go (null: nowhere)
__device__ __forceinline__ void store_row(bf16_t* dst, bf16_t* lo, const f32x16& a, float scale, int h) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint32_t w[4], r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = a[8 * j + 2 * i] * scale, y = a[8 * j + 2 * i + 1] * scale;
            w[i] = pack_bf16x2(x, y);
            r[i] = pack_bf16x2(x - __uint_as_float(w[i] << 16), y - __uint_as_float(w[i] & 0xffff0000u));
        }
        auto p0 = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false), p1 = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
        *reinterpret_cast<uint4*>(dst + 16 * j + 8 * h) = make_uint4(p0[0], p1[0], p0[1], p1[1]);
        if (lo) {
            p0 = __builtin_amdgcn_permlane32_swap(r[0], r[2], false, false); p1 = __builtin_amdgcn_permlane32_swap(r[1], r[3], false, false);
            *reinterpret_cast<uint4*>(lo + 16 * j + 8 * h) = make_uint4(p0[0], p1[0], p0[1], p1[1]);
        }
    }
}

// the same 32 channels in fp32, to a part
__device__ __forceinline__ void store_part(float* dst, const f32x16& a, float scale, int h) {
#pragma unroll
    for (int eg = 0; eg < 4; ++eg) *reinterpret_cast<float4*>(dst + 8 * eg + 4 * h) = make_float4(a[4 * eg] * scale, a[4 * eg + 1] * scale, a[4 * eg + 2] * scale, a[4 * eg + 3] * scale);
}

// ================================================================================================ forward
// 128 rows per workgroup of 4 waves, two workgroups per CU: one's softmax runs under the other's products without a barrier between them (8 waves of one workgroup: 3137 us where two
// of 4 take 2991; 64 rows a wave, one wave a SIMD: 3733; the next tile's S issued before this one's softmax within a wave: 3977).  16 + 16 products of 32 cycles a tile against
// ~300 vector instructions: the vector pipe is 40 - 49 % busy beside 40 - 57 % of the matrix pipe; at D = 64, with half the products, 47 beside 28.
// A sequence of 8 key tiles or fewer is bound by what a workgroup does once -- its sequence, its rows' loads, the stores: 6 of 22 us at 9216 queries on 512 keys.
// SPLIT, a few rows on long keys: HBM; 8 tokens on 60 354 keys, 32 / 8 heads of 128: 57 us = 4.3 TB/s from HBM, 42 us from the last-level cache.  Tiles of KR = 32 keys there, whose
// registers and LDS leave room for three workgroups a CU (tiles of 64, two: 6 % more), unless the parts are too few to fill them (2 tokens on 3000 keys: 16.3 us, with tiles of 64 15.8).
template <int D, bool SPLIT, int KR>
__global__ void __launch_bounds__(NT, KR == KT ? 2 : 3) varlen_fwd_kernel(const Params p) {
    constexpr int NKB = KR / 32, NKS = D / 16, NDB = D / 32, IMG = KR * D * 2, STAGE = 2 * IMG;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
    const Work w = find_work(blockIdx.x, p.hk, SPLIT ? p.nsplit : 1);
    const Tile t = find_tile<ROWS>(p, w.slot, false, p.causal);
    if (!t.live) return;

    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const Row r = find_row(p, t, w.head, wid, i);
    const Seen seen = keys_seen(p, t, wid);
    const bf16_t* K = p.k + t.k0 * p.k_ss + w.head * p.k_sh;
    const bf16_t* V = p.v + t.k0 * p.v_ss + w.head * p.v_sh;
    const bf16_t* Q = p.q + r.token * p.q_ss + r.head * p.q_sh;
    const float sl2 = p.scale * LOG2E;

    int kt0 = 0, kt1 = (seen.group + KR - 1) / KR;
    if (SPLIT) {                                               // every part of the sequence's key tiles, cut by its full length
        const int all = (t.lk + KR - 1) / KR, per = (all + p.nsplit - 1) / p.nsplit;
        kt0 = min(kt1, w.part * per); kt1 = min(kt1, kt0 + per);
    }
    Offsets<D, 4, KR> oK, oV;
    oK.init(wid, lane, p.k_ss); oV.init(wid, lane, p.v_ss);
    auto issue = [&](int kt) {
        char* base = lds + (kt & 1) * STAGE;
        oK.issue(rows_rsrc<D, KR>(K, p.k_ss, kt * KR, t.lk), base, wid);
        oV.issue(rows_rsrc<D, KR>(V, p.v_ss, kt * KR, t.lk), base + IMG, wid);
    };
    if (kt0 < kt1) issue(kt0);                                 // (in flight under the query's own loads)
    bf16x8_t qf[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qf[ks] = r.live ? *reinterpret_cast<const bf16x8_t*>(Q + 16 * ks + 8 * h) : zero_frag();
    f32x16 oacc[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) oacc[db] = zero16();
    float m = M_INIT, l = 0.f;                                 // running maximum in log2 units; this lane's part of the sum

    for (int kt = kt0; kt < kt1; ++kt) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // this wave's pieces of tile kt
        __builtin_amdgcn_s_barrier();                          // everyone's pieces landed; everyone is done with the other buffer
        if (kt + 1 < kt1) issue(kt + 1);
        const char* Kl = lds + (kt & 1) * STAGE;
        const char* Vl = Kl + IMG;
        const int key0 = kt * KR;
        if (key0 >= seen.wave) continue;                       // wave-uniform: no row of this wave sees the tile
        products_first<SPLIT ? 0 : D>(true);
        f32x16 s[NKB];
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) s[kb] = zero16();
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb) s[kb] = mfma16(by_rows<KR>(Kl, 32 * kb, ks, lane), qf[ks], s[kb]);
        products_first<SPLIT ? 0 : D>(false);
        if (key0 + KR > seen.all) {                            // some row of the wave does not see the whole tile
#pragma unroll
            for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[kb][e] = key0 + 32 * kb + (e & 3) + 8 * (e >> 2) + 4 * h <= r.last ? s[kb][e] : -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[kb][e]);
        mx = max_halves(mx) * sl2;
        if (!__all(mx <= m + RESCALE_AT)) {
            const float m_new = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - m_new);
            l *= alpha; m = m_new;
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
                for (int e = 0; e < 16; ++e) oacc[db][e] *= alpha;
        }
        float rs = 0.f;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) { const float pe = __builtin_amdgcn_exp2f(s[kb][e] * sl2 - m); s[kb][e] = pe; rs += pe; }
        l += rs;
        products_first<SPLIT ? 0 : D>(true);
#pragma unroll
        for (int u = 0; u < 2 * NKB; ++u) {                          // O^T += V^T . P^T, P rounded to the products' bf16
            const bf16x8_t pf = pack_frag(s[u >> 1], 8 * (u & 1));
#pragma unroll
            for (int db = 0; db < NDB; ++db) oacc[db] = mfma16(by_cols<KR>(Vl, 32 * db, 16 * u, lane), pf, oacc[db]);
        }
        if (key0 < KT) {                                       // the first 64 keys add what the rounding left (see CORNER)
#pragma unroll
            for (int u = 0; u < 2 * NKB; ++u) {
                const bf16x8_t pl = pack_rest(s[u >> 1], 8 * (u & 1));
#pragma unroll
                for (int db = 0; db < NDB; ++db) oacc[db] = mfma16(by_cols<KR>(Vl, 32 * db, 16 * u, lane), pl, oacc[db]);
            }
        }
    }

    const float sum = sum_halves(l);
    if (!r.live) return;
    const float inv = sum > 0.f ? 1.f / sum : sum;             // nothing seen: 0;  NaN stays NaN
    const float lse = sum == 0.f ? (SPLIT ? -INFINITY : INFINITY) : m + __builtin_amdgcn_logf(sum);      // v_log_f32 = log2
    const long row = r.token * p.hq + r.head, at = r.head * p.tq + r.token, part = SPLIT ? w.part * p.tq * p.hq : 0;
    if (h == 0 && (SPLIT || p.lse)) (SPLIT ? p.part_lse + part : p.lse)[at] = lse;
    if (SPLIT && sum == 0.f) return;                           // the join does not read this row
    if (r.last < 0) {                                          // sees no key: 0, also where its neighbours' keys are not finite
#pragma unroll
        for (int db = 0; db < NDB; ++db) oacc[db] = zero16();
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
        if (SPLIT) store_part(p.part + (part + row) * D + 32 * db, oacc[db], inv, h);
        else store_row(p.o + row * D + 32 * db, p.o_lo ? p.o_lo + row * D + 32 * db : nullptr, oacc[db], inv, h);
    }
}

// ================================================================================================ backward: dQ (and delta)
// 128 rows per workgroup, two workgroups per CU.  LDS operands four steps ahead of their products: 4050 -> 3956 us on the longest case above.  delta needs O to more than bf16 (dP and delta
// nearly cancel in dS): the forward keeps what the rounding of O left in bf16 too, 17 bits in 4 bytes a channel and half the traffic of an fp32 copy beside O (9216 queries on 512
// keys: forward 207 -> 169 us).
// Per 64-key tile: K, read by rows (S^T = K . Q^T) and transposed (dQ^T += K^T . dS^T), and V by rows (dP^T = V . dO^T).
template <int D, bool SPLIT>
__global__ void __launch_bounds__(NT, 2) varlen_dq_kernel(const Params p) {
    constexpr int NKS = D / 16, NDB = D / 32, IMG = KT * D * 2, STAGE = 2 * IMG;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
    const Work w = find_work(blockIdx.x, p.hk, SPLIT ? p.dq_split : 1);
    const Tile t = find_tile<ROWS>(p, w.slot, false, p.causal);
    if (!t.live) return;

    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const Row r = find_row(p, t, w.head, wid, i);
    const Seen seen = keys_seen(p, t, wid);
    const bf16_t* K = p.k + t.k0 * p.k_ss + w.head * p.k_sh;
    const bf16_t* V = p.v + t.k0 * p.v_ss + w.head * p.v_sh;
    const bf16_t* Q = p.q + r.token * p.q_ss + r.head * p.q_sh;
    const bf16_t* DO = p.dout + r.token * p.do_ss + r.head * p.do_sh;
    const long row = r.token * p.hq + r.head, at = r.head * p.tq + r.token;
    const float sl2 = p.scale * LOG2E;

    int kt0 = 0, nkt = (seen.group + KT - 1) / KT;
    if (SPLIT) {                                               // every part of the sequence's key tiles, cut by its full length
        const int all = (t.lk + KT - 1) / KT, per = (all + p.dq_split - 1) / p.dq_split;
        kt0 = min(nkt, w.part * per); nkt = min(nkt, kt0 + per);
    }
    Offsets<D, 4> oK, oV;
    oK.init(wid, lane, p.k_ss); oV.init(wid, lane, p.v_ss);
    auto issue = [&](int kt) {
        char* base = lds + (kt & 1) * STAGE;
        oK.issue(rows_rsrc<D>(K, p.k_ss, kt * KT, t.lk), base, wid);
        oV.issue(rows_rsrc<D>(V, p.v_ss, kt * KT, t.lk), base + IMG, wid);
    };
    if (kt0 < nkt) issue(kt0);
    // One tensor after the other: a load takes 32 bytes of 32 rows, the next three the rest of the same lines, which the L1 holds for four lines of a tensor a row but not for four
    // tensors' at once (with the four interleaved: 304 MB in 147 us instead of 66; the kernel at 9277 tokens, 32 heads 350 -> 335 us, at 9216 queries on 512 keys 270 -> 240).
    // A lane behind the last row reads the sequence's first: its P is 0 (lse), and nothing of its column is stored.
    bf16x8_t qf[NKS], dof[NKS], oh[NKS], ol[NKS];
    auto rows = [&](bf16x8_t (&f)[NKS], const bf16_t* src) {
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) f[ks] = *reinterpret_cast<const bf16x8_t*>(src + 16 * ks + 8 * h);
        __builtin_amdgcn_sched_barrier(0);
    };
    rows(qf, Q); rows(dof, DO); rows(oh, p.o + row * D); rows(ol, p.o_lo + row * D);
    float dl = 0.f;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks)
#pragma unroll
        for (int e = 0; e < 8; ++e) dl += (bf16_to_f32((bf16_t)oh[ks][e]) + bf16_to_f32((bf16_t)ol[ks][e])) * bf16_to_f32((bf16_t)dof[ks][e]);
    dl = sum_halves(dl);
    const float lse = r.live ? p.lse[at] : INFINITY;
    if (r.live && h == 0 && (!SPLIT || w.part == 0)) p.delta[at] = dl;
    f32x16 dq[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) dq[db] = zero16();

    for (int kt = kt0; kt < nkt; ++kt) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (kt + 1 < nkt) issue(kt + 1);
        const char* Kl = lds + (kt & 1) * STAGE;
        const char* Vl = Kl + IMG;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int key0 = kt * KT + 32 * kb;
            if (key0 >= seen.wave) break;
            f32x16 s = zero16(), dp = zero16();
            bf16x8_t f[AQ], kt[AQ];
            auto load = [&](int j) { return by_rows(j & 1 ? Vl : Kl, 32 * kb, j >> 1, lane); };
            auto load_t = [&](int j) { return by_cols(Kl, 32 * (j % NDB), 32 * kb + 16 * (j / NDB), lane); };
            products_first<D>(true);
            ahead_start(f, load);
            ahead_run<2 * NKS>(f, load, [&](int j, const bf16x8_t& x) { if (j & 1) dp = mfma16(x, dof[j >> 1], dp); else s = mfma16(x, qf[j >> 1], s); });
            ahead_start(kt, load_t);
            products_first<D>(false);
            if (key0 + 32 > seen.all) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = key0 + (e & 3) + 8 * (e >> 2) + 4 * h <= r.last ? s[e] : -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(s[e] * sl2 - lse) * (dp[e] - dl);
            if (key0 < KT) {                                   // (CORNER)
                const bf16x8_t rest[2] = {pack_rest(s, 0), pack_rest(s, 8)};
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int db = 0; db < NDB; ++db) dq[db] = mfma16(by_cols(Kl, 32 * db, 32 * kb + 16 * u, lane), rest[u], dq[db]);
            }
            const bf16x8_t ds[2] = {pack_frag(s, 0), pack_frag(s, 8)};
            products_first<D>(true);
            __builtin_amdgcn_sched_barrier(0);
            ahead_run<2 * NDB>(kt, load_t, [&](int j, const bf16x8_t& x) { dq[j % NDB] = mfma16(x, ds[j / NDB], dq[j % NDB]); });
        }
    }
    if (!r.live) return;
    if (r.last < 0) {                                          // sees no key: 0, whatever it and its gradient hold
#pragma unroll
        for (int db = 0; db < NDB; ++db) dq[db] = zero16();
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
        if (SPLIT) store_part(p.part + (w.part * p.tq * p.hq + row) * D + 32 * db, dq[db], p.scale, h); else store_row(p.dq + row * D + 32 * db, nullptr, dq[db], p.scale, h);
    }
}

// ================================================================================================ backward: dK, dV
// Key-outer; a lane owns one key column, K stays in LDS, V and both accumulators in registers:  S = Q . K^T, dP = dO . V^T, dV^T += dO^T . P, dK^T += Q^T . dS.  Per 64-query tile Q
// and dO, both read by rows and transposed, and the tile's lse / delta.  Query rows past the sequence arrive as zeros (Q, dO, lse, delta): P = 1 there, but dO = 0 and dS = 0.
// One kernel for dK and dV shares S and P between them (two kernels made 5 products instead of 4: 7764 -> 6134 us on the longest case above); K in LDS instead of registers gives the
// operands room one step ahead of their products (5992 -> 5640).  At D = 128 its 8 waves are two a SIMD and the LDS of a CU; 4 waves at D = 64, three a SIMD.
template <int D, int NW>
__global__ void __launch_bounds__(NW * 64, D == 64 ? 3 : 2) varlen_dkv_kernel(const Params p) {
    constexpr int QT = KT, NKS = D / 16, NDB = D / 32, IMG = QT * D * 2, O_STAT = 2 * IMG, STAGE = O_STAT + 1024;
    __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE + NW / 2 * IMG];
    const Work w = find_work(blockIdx.x, p.hk, p.nsplit);
    const Tile t = find_tile<32 * NW>(p, w.slot, true, false);
    if (!t.live) return;

    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const int k0w = (int)t.row0 + wid * 32, key = k0w + i;     // first key of this wave, this lane's key
    const bool live = key < t.lk;
    const int ahead = t.lk - t.lq;                             // causal: query x sees keys 0 .. x + ahead
    const float sl2 = p.scale * LOG2E;
    // query tiles: from the first one that sees a key of this workgroup, for each of the g heads; this part's share of them
    const int first = p.causal ? max(0, (int)t.row0 - ahead) / QT * QT : 0;
    const int per_head = max(0, (t.lq - first + QT - 1) / QT);
    const long all = (long)per_head * p.g, per = (all + p.nsplit - 1) / p.nsplit;
    const int twice = t.lq <= KT && t.lk <= KT ? 1 : 0;       // (CORNER) every tile once more, with what the rounding left
    const int it0 = (int)min(all, w.part * per), count = ((int)min(all, it0 + per) - it0) << twice;
    int hd = per_head > 0 ? it0 / per_head : 0, q = first + (it0 - hd * per_head) * QT;      // of the tile to fetch next
    const bf16_t* Q = p.q + t.q0 * p.q_ss + w.head * p.g * p.q_sh;
    const bf16_t* DO = p.dout + t.q0 * p.do_ss + w.head * p.g * p.do_sh;
    const long stat = (long)w.head * p.g * p.tq + t.q0;

    const char* Kl = lds + 2 * STAGE + wid / 2 * IMG;         // this wave's keys: rows 32 (wid & 1) .. of the image
    if (count > 0) {
        Offsets<D, NW> oK;
        oK.init(wid, lane, p.k_ss);
#pragma unroll
        for (int c = 0; c < NW / 2; ++c) oK.issue(rows_rsrc<D>(p.k + t.k0 * p.k_ss + w.head * p.k_sh, p.k_ss, (int)t.row0 + KT * c, t.lk), lds + 2 * STAGE + c * IMG, wid);
    }
    Offsets<D, NW> oQ, oD;
    oQ.init(wid, lane, p.q_ss); oD.init(wid, lane, p.do_ss);
    auto issue = [&](int buf) {
        char* base = lds + buf * STAGE;
        oQ.issue(rows_rsrc<D>(Q + hd * p.q_sh, p.q_ss, q, t.lq), base, wid);
        oD.issue(rows_rsrc<D>(DO + hd * p.do_sh, p.do_ss, q, t.lq), base + IMG, wid);
        const int bytes = min(QT, t.lq - q) * 4;
        if (wid == 0) dma4(tile_rsrc(p.lse + stat + hd * p.tq + q, bytes), base + O_STAT, lane * 4);
        if (wid == 1) dma4(tile_rsrc(p.delta + stat + hd * p.tq + q, bytes), base + O_STAT + 256, lane * 4);
    };
    if (count > 0) issue(0);
    const bf16_t* V = p.v + (t.k0 + (live ? key : 0)) * p.v_ss + w.head * p.v_sh;
    bf16x8_t vf[NKS];
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) vf[ks] = live ? *reinterpret_cast<const bf16x8_t*>(V + 16 * ks + 8 * h) : zero_frag();
    f32x16 dk[NDB], dv[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) { dk[db] = zero16(); dv[db] = zero16(); }
    for (int it = 0; it < count; ++it) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        const int qt = q;                                      // the tile at hand
        const bool rest = twice & it;
        if (!twice || rest) {
            q += QT;
            if (q >= t.lq) { q = first; ++hd; }
        }
        if (it + 1 < count) issue((it + 1) & 1);
        const char* Ql = lds + (it & 1) * STAGE;
        const char* DOl = Ql + IMG;
        const float* lse_l = reinterpret_cast<const float*>(Ql + O_STAT);
        const float* dl_l = lse_l + QT;
        if (k0w >= t.lk) continue;                             // wave-uniform: no live key
#pragma unroll
        for (int qb = 0; qb < 2; ++qb) {
            const int q0 = qt + 32 * qb;
            if (q0 >= t.lq) break;
            if (p.causal && q0 + 31 + ahead < k0w) continue;   // no query of the block sees a key of this wave
            f32x16 s = zero16(), dp = zero16();
            struct Frags { bf16x8_t q, d, k; };
            Frags f[AK], g[AK];
            auto load = [&](int j) { return Frags{by_rows(Ql, 32 * qb, j, lane), by_rows(DOl, 32 * qb, j, lane), by_rows(Kl, 32 * (wid & 1), j, lane)}; };
            auto load_t = [&](int j) {
                return Frags{by_cols(Ql, 32 * (j % NDB), 32 * qb + 16 * (j / NDB), lane), by_cols(DOl, 32 * (j % NDB), 32 * qb + 16 * (j / NDB), lane), {}};
            };
            products_first<D>(true);
            ahead_start(f, load);
            ahead_run<NKS>(f, load, [&](int j, const Frags& x) { s = mfma16(x.q, x.k, s); dp = mfma16(x.d, vf[j], dp); });
            ahead_start(g, load_t);
            products_first<D>(false);
            if (p.causal && q0 + ahead < k0w + 31) {           // some query of the block does not see every key of this wave
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = key <= q0 + 8 * (e >> 2) + 4 * h + (e & 3) + ahead ? s[e] : -INFINITY;
            }
            f32x16 pr;
#pragma unroll
            for (int eg = 0; eg < 4; ++eg) {
                const float4 l4 = *reinterpret_cast<const float4*>(&lse_l[32 * qb + 8 * eg + 4 * h]), d4 = *reinterpret_cast<const float4*>(&dl_l[32 * qb + 8 * eg + 4 * h]);
                const float ll[4] = {l4.x, l4.y, l4.z, l4.w}, dd[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = 4 * eg + j;
                    pr[e] = __builtin_amdgcn_exp2f(s[e] * sl2 - ll[j]);
                    s[e] = pr[e] * (dp[e] - dd[j]);
                }
            }
            if (rest) { rounding_left(pr); rounding_left(s); }
            const bf16x8_t pf[2] = {pack_frag(pr, 0), pack_frag(pr, 8)}, ds[2] = {pack_frag(s, 0), pack_frag(s, 8)};
            products_first<D>(true);
            __builtin_amdgcn_sched_barrier(0);
            ahead_run<2 * NDB>(g, load_t, [&](int j, const Frags& x) { dv[j % NDB] = mfma16(x.d, pf[j / NDB], dv[j % NDB]); dk[j % NDB] = mfma16(x.q, ds[j / NDB], dk[j % NDB]); });
        }
    }
    if (!live) return;
    const long row = ((t.k0 + key) * p.hk + w.head) * D, slice = p.tk * p.hk * D;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
        if (p.nsplit == 1) {
            store_row(p.dk + row + 32 * db, nullptr, dk[db], p.scale, h);
            store_row(p.dv + row + 32 * db, nullptr, dv[db], 1.f, h);
            continue;
        }
#pragma unroll
        for (int eg = 0; eg < 4; ++eg) {
            const long at = row + 32 * db + 8 * eg + 4 * h;
            *reinterpret_cast<float4*>(p.part + 2 * w.part * slice + at) = make_float4(dk[db][4 * eg] * p.scale, dk[db][4 * eg + 1] * p.scale, dk[db][4 * eg + 2] * p.scale, dk[db][4 * eg + 3] * p.scale);
            *reinterpret_cast<float4*>(p.part + (2 * w.part + 1) * slice + at) = make_float4(dv[db][4 * eg], dv[db][4 * eg + 1], dv[db][4 * eg + 2], dv[db][4 * eg + 3]);
        }
    }
}

// ------------------------------------------------------------------------------------------------ host side
// In how many parts (own workgroups, fp32 partial results, a kernel that sums them) an axis is cut that workgroups walk in LDS tiles: the least of the estimated times
//   us(parts) = tile * tiles / parts * max(longest, share * x) + once * x / per_cu + (parts > 1: sum + part * parts),    x = workgroups per CU
// tile: a tile's time for a workgroup that has its CU to itself; share: what of it is left per workgroup when several share the CU; once: a workgroup's start and end; sum, part: the
// kernel that sums, and what a part adds.  One sequence: its tiles, and x rounded up (all its workgroups take the same time).  Several: the lengths are on the device, so the average's
// tiles, the longest taken as 1.5 of it, their rows as one sequence's but for `once`, with at least a workgroup a sequence and head; and of the cuts within 10 % the finest, which
// balances best.  Measured, with the sums, us, whole / as chosen.  Forward: 8 tokens on 3 x 10 000 keys, 12 / 4 heads of 64: 240 / 17; 4096 tokens, 4 heads of 128: 84 / 61, 7 heads
// 89 / 89 (four parts 102); 2048 tokens, 12 heads of 64: 33 / 33 (three parts 45); 8000 queries on 512 keys, 4 heads: 21 / 21 (three parts 49).  dK / dV: 1000 tokens, 10 heads: 52 / 41;
// 4096 tokens, 4 heads 190 / 94, 7 heads 198 / 147; 8000 queries on 512 keys 346 / 44; six causal sequences of 1000, 8 heads: 60 / 60 (three parts 94).
// The average says nothing about one sequence among many: offsets of a fixed capacity end in empty sequences, and a long one may have short neighbours.  The other extreme is one
// sequence that holds all rows and the whole axis, beside workgroups that find nothing to do (1 ns a sequence, head and part; a quarter where there are more sequences than rows).  The
// parts are the fewest, from the average's choice on, that are estimated at no more than twice the least time there.  By the average alone / as chosen, us a replayed call, 32 / 8 heads
// of 128: 1 row on 8191 keys in offsets for 64 sequences 146 / 53 (for one 22), 64 rows on 30 063 keys in offsets for 64 527 / 141 (61), 64 single tokens, one on 16 384 keys and 63 on
// 100, 284 / 92; 4 heads, forward and backward: 8000 queries on 512 keys in offsets for 16 403 / 132 (91), 4096 + 15 x 64 causal tokens 370 / 296.  What equal lengths pay for it: 64
// single tokens on 512 keys each 29 / 39, on 2048 113 / 124, 16 on 512 18 / 20; longer rows nothing (12 x 1000 tokens, 8 heads, 242 / 242).
struct SplitCost { float tile, share, once, sum, part; int per_cu; };
int best_parts(long row_tiles, long rows, int heads, long tiles, long all_tiles, int n, const SplitCost& k) {      // tiles: a sequence's on average; all_tiles: the whole axis
    const float cu = heads / 256.f, groups = row_tiles > n ? row_tiles : n < rows ? n : rows, idle = 1e-3f * heads * (n < rows ? n : 0.25f * n + 0.75f * rows);
    auto us = [&](int s) {
        const float x = n > 1 ? row_tiles * s * cu : ceilf(row_tiles * s * cu);
        return k.tile * tiles / s * fmaxf(n > 1 ? 1.5f : 1.f, k.share * x) + k.once * ceilf(groups * s * cu / k.per_cu) + (s > 1 ? k.sum + k.part * s : 0.f);
    };
    auto us_one = [&](int s) {
        const float x = ceilf(row_tiles * s * cu);
        return k.tile * all_tiles / s * fmaxf(1.f, k.share * x) + k.once * ceilf(row_tiles * s * cu / k.per_cu) + (s > 1 ? k.sum + k.part * s : 0.f) + idle * s;
    };
    auto most = [](long t) { return t < 8 ? 1 : t < 128 ? (int)t / 2 : 64; };      // at least two tiles a part
    int best = 1;
    for (int s = 2; s <= most(tiles); ++s) if (us(s) < us(best)) best = s;
    if (n == 1) return best;
    if (best > 1) {
        const float close = 1.1f * us(best);
        for (int s = most(tiles); s > best; --s) if (us(s) <= close) { best = s; break; }
    }
    float least = us_one(1);
    for (int s = 2; s <= most(all_tiles); ++s) least = fminf(least, us_one(s));
    while (best < most(all_tiles) && us_one(best) > 2.f * least) ++best;
    return best;
}
// no more parts than leave the grid below 2^23 workgroups
constexpr long MAX_GROUPS = (1l << 23) - 1;
int fitting(long parts, long slots, int heads) { const long most = MAX_GROUPS / work_groups(slots, heads, 1); return (int)(parts > most && parts > 1 ? (most > 1 ? most : 1) : parts); }
// parts of the key range, D = 128 / 64: 1.2 / 0.85 us a tile (a workgroup's run over 64 tiles alone on its CU: 84 us, two to a CU 1.9 us a tile each)
int fwd_splits(long tq, long tk, int n, int hq, int hk, int D) {
    const float m = tq * hq * (float)D * 1e-6f;               // (millions of partial results a part)
    const long rows = tq * (hq / hk);
    const int s = best_parts(cdiv(rows, ROWS), rows, hk, tk / n / KT, tk / KT, n, {D == 128 ? 1.2f : 0.85f, D == 128 ? 0.78f : 0.55f, 7.f, 5.5f + 2.5f * m, 1.5f * m, D == 128 ? 2 : 3});
    return fitting(s, rows / ROWS + n + 1, hk);
}
// keys of a dK / dV workgroup: 8 waves at D = 128, whose K image and registers leave room for one workgroup per CU, 4 at 64
constexpr int key_tile(int D) { return D == 128 ? 256 : 128; }
// parts of the key range for dQ, D = 128 / 64: 1.55 / 1.2 us a tile.  With the sum, us, whole / as chosen: 4096 tokens, 4 heads
// of 128: 106 / 76; 500 queries on 4000 + 3000 keys, 8 heads: 98 / 43; 3000 causal tokens, 3 / 1 heads of 64: 54 / 28; 2048 tokens, 10 heads of 128: 58 / 58
int dq_splits(long tq, long tk, int n, int hq, int hk, int D) {
    const long rows = tq * (hq / hk);
    const int s = best_parts(cdiv(rows, ROWS), rows, hk, tk / n / KT, tk / KT, n, {D == 128 ? 1.55f : 1.2f, D == 128 ? 0.94f : 0.75f, 8.f, 6.f, 1.6f * (tq * hq * (float)D * 1e-6f), D == 128 ? 2 : 3});
    return fitting(s, rows / ROWS + n + 1, hk);
}
// parts of the query tiles (of all g heads) for dK / dV, D = 128 / 64: 3.0 / 1.6 us a tile.  With grouped heads up to g parts also where the key tiles alone are fewer than 3 a CU and the
// sequences long enough that the parts' fp32 sums do not cost more than the balance gives (4 x 2048 causal tokens, 32 / 8 heads, backward: 648 -> 604 us; 16 x 512: 310 unsplit, 332 split)
int dkv_splits(long tq, long tk, int n, int hq, int hk, int D) {
    const long key_tiles = cdiv(tk, key_tile(D)), wgs = key_tiles * hk, g = hq / hk, tiles = tq / n / KT * g;
    const float part = 3.1f * (tk * hk * (float)D * 1e-6f);
    long s = D == 128 ? best_parts(key_tiles, tk, hk, tiles, tq / KT * g, n, {3.0f, 1.0f, 6.f, 6.f, part, 1}) : best_parts(key_tiles, tk, hk, tiles, tq / KT * g, n, {1.6f, 0.55f, 6.f, 6.f, part, 3});
    if (wgs < 768 && g > 1 && tiles >= 16 * g) { long m = cdiv(768, wgs); if (m > g) m = g; if (m > s) s = m; }
    return fitting(s > 64 ? 64 : s, tk / ROWS + n + 1, hk);
}

bool rows_ok(const void* p, long ss, long sh, int D) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ss % 8 == 0 && sh % 8 == 0 && ss >= D && ss < (1l << 23) && sh >= 0;
}

template <typename T>
int fill(VarlenParams<T>& p, const char* what, const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, long tq, long tk, int n, int hq, int hk, int D, long q_ss,
         long q_sh, long k_ss, long k_sh, long v_ss, long v_sh, float scale, int causal, bool backward) {
    auto bad = [&](const char* m, int rc = DPIPE_ERR_ARG) { char buf[160]; snprintf(buf, sizeof(buf), "%s: %s", what, m); set_last_error(buf); return rc; };
    if (!q || !k || !v || !cu_q || !cu_k || tq <= 0 || tk <= 0 || n <= 0 || hq <= 0 || hk <= 0 || hq % hk) return bad("bad argument");
    if (D != 64 && D != 128) return bad("head dim must be 64 or 128", DPIPE_ERR_UNSUPPORTED);
    if (!(scale > 0.f) || scale > 1e30f) return bad("scale must be positive and finite");
    p.nsplit = backward ? dkv_splits(tq, tk, n, hq, hk, D) : fwd_splits(tq, tk, n, hq, hk, D);
    p.dq_split = backward ? dq_splits(tq, tk, n, hq, hk, D) : 1;
    if (tq * (hq / hk) >= (1l << 31) - 256 || tk >= (1l << 31) - 256 || work_groups(tq * (hq / hk) / ROWS + n + 1, hk, backward ? p.dq_split : p.nsplit) > MAX_GROUPS ||
        (backward && work_groups(tk / ROWS + n + 1, hk, p.nsplit) > MAX_GROUPS))
        return bad("too many rows or sequences", DPIPE_ERR_UNSUPPORTED);
    if (!rows_ok(q, q_ss, q_sh, D) || !rows_ok(k, k_ss, k_sh, D) || !rows_ok(v, v_ss, v_sh, D)) return bad("tensors must be 16-byte aligned with strides multiple of 8 elements");
    p.q = (const T*)q; p.k = (const T*)k; p.v = (const T*)v; p.cu_q = cu_q; p.cu_k = cu_k; p.tq = tq; p.tk = tk; p.n = n; p.hq = hq; p.hk = hk; p.g = hq / hk;
    p.q_ss = q_ss; p.q_sh = q_sh; p.k_ss = k_ss; p.k_sh = k_sh; p.v_ss = v_ss; p.v_sh = v_sh; p.scale = scale; p.causal = causal != 0;
    return DPIPE_OK;
}

template <int D> void forward(const Params& p, hipStream_t s) {
    const unsigned grid = (unsigned)work_groups(row_slots(p.tq, p.g, p.n, ROWS), p.hk, p.nsplit);
    if (p.nsplit == 1) { varlen_fwd_kernel<D, false, KT><<<grid, NT, 0, s>>>(p); return; }
    if (D == 128 && p.nsplit * (cdiv(p.tq * p.g, ROWS) + p.n - 1) * p.hk >= 512) varlen_fwd_kernel<D, true, D == 128 ? 32 : KT><<<grid, NT, 0, s>>>(p);
    else varlen_fwd_kernel<D, true, KT><<<grid, NT, 0, s>>>(p);
    join<bf16_t, D>(p, s);
}
template <int D> void backward(const Params& p, hipStream_t s) {
    const unsigned rows = (unsigned)work_groups(row_slots(p.tq, p.g, p.n, ROWS), p.hk, p.dq_split);
    if (p.dq_split == 1) varlen_dq_kernel<D, false><<<rows, NT, 0, s>>>(p);
    else { varlen_dq_kernel<D, true><<<rows, NT, 0, s>>>(p); sum_parts(p, p.dq, (bf16_t*)nullptr, p.dq_split, p.tq * p.hq * D, s); }
    constexpr int NW = key_tile(D) / 32;
    const unsigned keys = (unsigned)work_groups(row_slots(p.tk, 1, p.n, 32 * NW), p.hk, p.nsplit);
    varlen_dkv_kernel<D, NW><<<keys, 64 * NW, 0, s>>>(p);
    if (p.nsplit > 1) sum_parts(p, p.dk, p.dv, p.nsplit, p.tk * p.hk * D, s);
}
// fp32 values of the parts: dQ's are summed before dK's and dV's are written
long bwd_floats(long tq, long tk, int hq, int hk, int D, int dq_parts, int dkv_parts) {
    const long a = dq_parts > 1 ? dq_parts * tq * hq * D : 0, b = dkv_parts > 1 ? 2l * dkv_parts * tk * hk * D : 0;
    return a > b ? a : b;
}

}  // namespace

extern "C" {

long dpipe_attn_varlen_fwd_workspace_floats(long tq, long tk, int n, int hq, int hk, int D) {
    if (tq <= 0 || tk <= 0 || n <= 0 || hq <= 0 || hk <= 0 || hq % hk || (D != 64 && D != 128)) return 0;
    const int s = fwd_splits(tq, tk, n, hq, hk, D);
    return s > 1 ? (long)s * tq * hq * (D + 1) : 0;
}
long dpipe_attn_varlen_bwd_workspace_floats(long tq, long tk, int n, int hq, int hk, int D) {
    if (tq <= 0 || tk <= 0 || n <= 0 || hq <= 0 || hk <= 0 || hq % hk || (D != 64 && D != 128)) return 0;
    return bwd_floats(tq, tk, hq, hk, D, dq_splits(tq, tk, n, hq, hk, D), dkv_splits(tq, tk, n, hq, hk, D));
}

int dpipe_attn_varlen_fwd(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, void* o, void* o_lo, float* lse, float* ws, long ws_floats, long tq,
                          long tk, int n, int hq, int hk, int D, long q_ss, long q_sh, long k_ss, long k_sh, long v_ss, long v_sh, float scale, int causal, int dtype, void* stream) {
    auto run = [&](auto type, auto launch) {
        typedef decltype(type) T;
        VarlenParams<T> p = {};
        const int rc = fill(p, "dpipe_attn_varlen_fwd", q, k, v, cu_q, cu_k, tq, tk, n, hq, hk, D, q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, scale, causal, false);
        if (rc) return rc;
        const long need = p.nsplit > 1 ? (long)p.nsplit * tq * hq * (D + 1) : 0;
        if (!o || !aligned16(o) || !aligned16(o_lo) || (need > 0 && (!ws || ws_floats < need || !aligned16(ws)))) {
            set_last_error("dpipe_attn_varlen_fwd: bad output or workspace"); return DPIPE_ERR_ARG; }
        if (ablated(ABL_ATTN)) return DPIPE_OK;
        p.o = (T*)o; p.o_lo = sizeof(T) == 2 ? (T*)o_lo : nullptr; p.lse = lse;
        if (need > 0) { p.part = ws; p.part_lse = ws + (long)p.nsplit * tq * hq * D; }
        launch(p);
        return check_launch("dpipe_attn_varlen_fwd");
    };
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == DPIPE_BF16) return run(bf16_t{}, [&](auto& p) { if (D == 64) forward<64>(p, s); else forward<128>(p, s); });
    if (dtype == DPIPE_F32) return run(float{}, [&](auto& p) { forward_f32(p, D, s); });
    set_last_error("dpipe_attn_varlen_fwd: dtype must be bf16 or fp32");
    return DPIPE_ERR_UNSUPPORTED;
}

int dpipe_attn_varlen_bwd(const void* q, const void* k, const void* v, const int* cu_q, const int* cu_k, const void* o, const void* o_lo, const void* dout, const float* lse, float* delta,
                          void* dq, void* dk, void* dv, float* ws, long ws_floats, long tq, long tk, int n, int hq, int hk, int D, long q_ss, long q_sh, long k_ss, long k_sh,
                          long v_ss, long v_sh, long do_ss, long do_sh, float scale, int causal, int dtype, void* stream) {
    auto run = [&](auto type, auto launch) {
        typedef decltype(type) T;
        VarlenParams<T> p = {};
        const int rc = fill(p, "dpipe_attn_varlen_bwd", q, k, v, cu_q, cu_k, tq, tk, n, hq, hk, D, q_ss, q_sh, k_ss, k_sh, v_ss, v_sh, scale, causal, true);
        if (rc) return rc;
        const long need = bwd_floats(tq, tk, hq, hk, D, p.dq_split, p.nsplit);
        if (!o || (sizeof(T) == 2 && !o_lo) || !dout || !lse || !delta || !dq || !dk || !dv || !aligned16(o) || !aligned16(o_lo) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv) ||
            !rows_ok(dout, do_ss, do_sh, D) || (need > 0 && (!ws || ws_floats < need || !aligned16(ws)))) {
            set_last_error("dpipe_attn_varlen_bwd: bad gradient or workspace"); return DPIPE_ERR_ARG; }
        if (ablated(ABL_ATTN)) return DPIPE_OK;
        p.o = (T*)o; p.o_lo = (T*)o_lo; p.dout = (const T*)dout; p.lse = const_cast<float*>(lse); p.delta = delta;
        p.dq = (T*)dq; p.dk = (T*)dk; p.dv = (T*)dv; p.do_ss = do_ss; p.do_sh = do_sh; p.part = ws;
        launch(p);
        return check_launch("dpipe_attn_varlen_bwd");
    };
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    if (dtype == DPIPE_BF16) return run(bf16_t{}, [&](auto& p) { if (D == 64) backward<64>(p, s); else backward<128>(p, s); });
    if (dtype == DPIPE_F32) return run(float{}, [&](auto& p) { backward_f32(p, D, s); });
    set_last_error("dpipe_attn_varlen_bwd: dtype must be bf16 or fp32");
    return DPIPE_ERR_UNSUPPORTED;
}

}  // extern "C"
