// attention_varlen_f32.hip -- the fp32 form of attention_varlen.hip (same contract, same tiles of 128 rows and same parts), for runs that keep every product in fp32: v_mfma_f32_32x32x2_f32.
//
// The transposed score tile again: entry e of lane (i, h) is key (dK / dV: query) 4 h + (e & 3) + 8 (e >> 2) of column i, which is just the B operand of a two-deep product whose k slot
// h is that row -- P and dS go back into the matrix pipe straight from their accumulators, one entry a product.  Tiles of 32 rows, staged through registers into LDS (a bound check
// fills the rows past a sequence with zeros); the row pitch of D + 2 floats makes the row reads (8 bytes a lane) conflict-free, and a product of 64 cycles hides them.
//
// Bound: the fp32 matrix pipe, 1 / 16 of the bf16 rate (an 8192^3 library product: 153 TFLOP/s).  1311 + 2560 + 4608 tokens, 24 heads of 128: forward 2.92 ms = 124 TFLOP/s, dQ 4.38 ms
// = 124, dK / dV 6.73 ms = 108; 8 x 1024 tokens, 24 heads of 64: 0.43 / 0.61 / 0.85 ms.  (The axes are cut by the estimate of the bf16 kernels.)  What hides the staging is measured per kernel: the next tile's loads in flight over this one's
// products (forward 4.70 -> 3.23 ms, backward 14.6 -> 11.5), then two workgroups to a CU where 256 registers a lane are enough (forward 3.23 -> 2.95); dQ at D = 128 has them with no
// loads ahead (4.38 - 4.59 ms, 22 registers spilled, 10 scratch accesses beside a tile's 192 products; one workgroup with loads ahead 4.68), dK / dV at D = 128 keeps K, V, dK and dV of 32 keys in registers and has one.
#include "dpipe_common.h"
#include "attention_tiles.h"
#include "attention_varlen.h"

using namespace dpipe;
using namespace dpipe_tiles;
using namespace dpipe_varlen;

namespace {

typedef VarlenParams<float> Params;
constexpr int KT = 32;                   // rows of a staged tile

__device__ __forceinline__ f32x16 mfma2(float a, float b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
__device__ __forceinline__ int entry_row(int e, int h) { return (e & 3) + 8 * (e >> 2) + 4 * h; }

// Rows at .. at + 31 (zero from n on) of a [*, D] matrix with row pitch ss, on their way into LDS: the next tile's loads are in flight while this one's is multiplied.
template <int D> struct Staged {
    static constexpr int N = KT * D / 4 / NT;
    float4 v[N];
    __device__ __forceinline__ void load(const float* base, long ss, int at, int n) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int x = threadIdx.x + j * NT, row = x / (D / 4), c = 4 * (x % (D / 4));
            v[j] = at + row < n ? *reinterpret_cast<const float4*>(base + (long)(at + row) * ss + c) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    __device__ __forceinline__ void store(float* dst) const {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int x = threadIdx.x + j * NT, row = x / (D / 4), c = 4 * (x % (D / 4));
            *reinterpret_cast<float2*>(dst + row * (D + 2) + c) = make_float2(v[j].x, v[j].y);
            *reinterpret_cast<float2*>(dst + row * (D + 2) + c + 2) = make_float2(v[j].z, v[j].w);
        }
    }
};
// a row's channels 4 j + 2 h, + 1 in the lane: its operand of the products over channels
template <int D> struct RowOperand {
    float2 v[D / 4];
    __device__ __forceinline__ void load(const float* row, int h, bool live) {
#pragma unroll
        for (int j = 0; j < D / 4; ++j) v[j] = live ? *reinterpret_cast<const float2*>(row + 4 * j + 2 * h) : make_float2(0.f, 0.f);
    }
};
// tile . operand^T over the channels: a 32 x 32 score tile
template <int D> __device__ __forceinline__ f32x16 over_channels(const float* tile, const RowOperand<D>& x, int lane) {
    f32x16 s = zero16();
    const float* r = tile + (lane & 31) * (D + 2) + 2 * (lane >> 5);
#pragma unroll
    for (int j = 0; j < D / 4; ++j) {
        const float2 a = *reinterpret_cast<const float2*>(r + 4 * j);
        s = mfma2(a.x, x.v[j].x, s); s = mfma2(a.y, x.v[j].y, s);
    }
    return s;
}
// acc += tile^T . s over the tile's rows
template <int D> __device__ __forceinline__ void over_rows(f32x16* acc, const float* tile, const f32x16& s, int lane) {
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
        for (int db = 0; db < D / 32; ++db) acc[db] = mfma2(tile[entry_row(e, lane >> 5) * (D + 2) + 32 * db + (lane & 31)], s[e], acc[db]);
}
__device__ __forceinline__ void store_row(float* dst, const f32x16& a, float scale, int h) {
#pragma unroll
    for (int eg = 0; eg < 4; ++eg) *reinterpret_cast<float4*>(dst + 8 * eg + 4 * h) = make_float4(a[4 * eg] * scale, a[4 * eg + 1] * scale, a[4 * eg + 2] * scale, a[4 * eg + 3] * scale);
}

template <int D, bool SPLIT>
__global__ void __launch_bounds__(NT, 2) varlen_f32_fwd_kernel(const Params p) {
    constexpr int NDB = D / 32;
    __shared__ __attribute__((aligned(16))) float Kl[KT * (D + 2)], Vl[KT * (D + 2)];
    const Work w = find_work(blockIdx.x, p.hk, SPLIT ? p.nsplit : 1);
    const Tile t = find_tile<ROWS>(p, w.slot, false, p.causal);
    if (!t.live) return;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const Row r = find_row(p, t, w.head, wid, i);
    const Seen seen = keys_seen(p, t, wid);
    const float sl2 = p.scale * LOG2E;
    RowOperand<D> q;
    q.load(p.q + r.token * p.q_ss + r.head * p.q_sh, h, r.live);
    f32x16 o[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[db] = zero16();
    float m = M_INIT, l = 0.f;
    int k0 = 0, k1 = seen.group;
    if (SPLIT) {                                               // every part of the sequence's key tiles, cut by its full length
        const int per = ((t.lk + KT - 1) / KT + p.nsplit - 1) / p.nsplit * KT;
        k0 = min((long)k1, (long)w.part * per); k1 = min(k1, k0 + per);
    }
    const float *kp = p.k + t.k0 * p.k_ss + w.head * p.k_sh, *vp = p.v + t.k0 * p.v_ss + w.head * p.v_sh;
    Staged<D> ks, vs;
    ks.load(kp, p.k_ss, k0, k1); vs.load(vp, p.v_ss, k0, k1);
    for (int key0 = k0; key0 < k1; key0 += KT) {
        __syncthreads();
        ks.store(Kl); vs.store(Vl);
        __syncthreads();
        ks.load(kp, p.k_ss, key0 + KT, k1); vs.load(vp, p.v_ss, key0 + KT, k1);
        if (key0 >= seen.wave) continue;                       // wave-uniform
        f32x16 s = over_channels<D>(Kl, q, lane);
        float mx = -INFINITY;
#pragma unroll
        for (int e = 0; e < 16; ++e) { s[e] = key0 + entry_row(e, h) <= r.last ? s[e] : -INFINITY; mx = fmaxf(mx, s[e]); }
        mx = max_halves(mx) * sl2;
        if (!__all(mx <= m + RESCALE_AT)) {
            const float m_new = fmaxf(m, mx), alpha = __builtin_amdgcn_exp2f(m - m_new);
            l *= alpha; m = m_new;
#pragma unroll
            for (int db = 0; db < NDB; ++db)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[db][e] *= alpha;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) { s[e] = __builtin_amdgcn_exp2f(s[e] * sl2 - m); l += s[e]; }
        over_rows<D>(o, Vl, s, lane);
    }
    const float sum = sum_halves(l);
    if (!r.live) return;
    const float inv = sum > 0.f ? 1.f / sum : sum;             // nothing seen: 0;  NaN stays NaN
    const long row = r.token * p.hq + r.head, at = r.head * p.tq + r.token, part = SPLIT ? w.part * p.tq * p.hq : 0;
    const float lse = sum == 0.f ? (SPLIT ? -INFINITY : INFINITY) : m + __builtin_amdgcn_logf(sum);
    if (h == 0 && (SPLIT || p.lse)) (SPLIT ? p.part_lse + part : p.lse)[at] = lse;
    if (SPLIT && sum == 0.f) return;
    if (r.last < 0) {                                          // sees no key: 0, also where its neighbours' keys are not finite
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db] = zero16();
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) store_row((SPLIT ? p.part + part * D : p.o) + row * D + 32 * db, o[db], inv, h);
}

template <int D, bool SPLIT>
__global__ void __launch_bounds__(NT, 2) varlen_f32_dq_kernel(const Params p) {
    constexpr int NDB = D / 32;
    __shared__ __attribute__((aligned(16))) float Kl[KT * (D + 2)], Vl[KT * (D + 2)];
    const Work w = find_work(blockIdx.x, p.hk, SPLIT ? p.dq_split : 1);
    const Tile t = find_tile<ROWS>(p, w.slot, false, p.causal);
    if (!t.live) return;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const Row r = find_row(p, t, w.head, wid, i);
    const Seen seen = keys_seen(p, t, wid);
    const float sl2 = p.scale * LOG2E;
    const long row = r.token * p.hq + r.head, at = r.head * p.tq + r.token;
    RowOperand<D> q, d;
    d.load(p.dout + r.token * p.do_ss + r.head * p.do_sh, h, r.live);
    float dl = 0.f;                                            // delta = rowsum(dO . O)
#pragma unroll
    for (int j = 0; j < D / 4; ++j) {
        const float2 o = *reinterpret_cast<const float2*>(p.o + row * D + 4 * j + 2 * h);       // (a lane without a row reads its sequence's first: its dO is 0 -- delta may be NaN, unused)
        dl += d.v[j].x * o.x + d.v[j].y * o.y;
    }
    q.load(p.q + r.token * p.q_ss + r.head * p.q_sh, h, r.live);
    dl = sum_halves(dl);
    const float lse = r.live ? p.lse[at] : INFINITY;
    if (r.live && h == 0 && (!SPLIT || w.part == 0)) p.delta[at] = dl;
    f32x16 dq[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) dq[db] = zero16();
    int k0 = 0, k1 = seen.group;
    if (SPLIT) {
        const int per = ((t.lk + KT - 1) / KT + p.dq_split - 1) / p.dq_split * KT;
        k0 = min((long)k1, (long)w.part * per); k1 = min(k1, k0 + per);
    }
    const float *kp = p.k + t.k0 * p.k_ss + w.head * p.k_sh, *vp = p.v + t.k0 * p.v_ss + w.head * p.v_sh;
    Staged<D> ks, vs;
    constexpr bool AHEAD = D == 64;                            // (D = 128: the other workgroup of the CU computes meanwhile)
    if (AHEAD) { ks.load(kp, p.k_ss, k0, k1); vs.load(vp, p.v_ss, k0, k1); }
    for (int key0 = k0; key0 < k1; key0 += KT) {
        if (!AHEAD) { ks.load(kp, p.k_ss, key0, k1); vs.load(vp, p.v_ss, key0, k1); }
        __syncthreads();
        ks.store(Kl); vs.store(Vl);
        __syncthreads();
        if (AHEAD) { ks.load(kp, p.k_ss, key0 + KT, k1); vs.load(vp, p.v_ss, key0 + KT, k1); }
        if (key0 >= seen.wave) continue;
        f32x16 s = over_channels<D>(Kl, q, lane);
        const f32x16 dp = over_channels<D>(Vl, d, lane);
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = key0 + entry_row(e, h) <= r.last ? __builtin_amdgcn_exp2f(s[e] * sl2 - lse) * (dp[e] - dl) : 0.f;
        over_rows<D>(dq, Kl, s, lane);
    }
    if (!r.live) return;
    if (r.last < 0) {
#pragma unroll
        for (int db = 0; db < NDB; ++db) dq[db] = zero16();
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db) store_row((SPLIT ? p.part + w.part * p.tq * p.hq * D : p.dq) + row * D + 32 * db, dq[db], p.scale, h);
}

template <int D>
__global__ void __launch_bounds__(NT, D == 64 ? 2 : 1) varlen_f32_dkv_kernel(const Params p) {
    constexpr int NDB = D / 32;
    __shared__ __attribute__((aligned(16))) float Ql[KT * (D + 2)], DOl[KT * (D + 2)], stat[2][KT];
    const Work w = find_work(blockIdx.x, p.hk, p.nsplit);
    const Tile t = find_tile<ROWS>(p, w.slot, true, false);
    if (!t.live) return;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 31, h = lane >> 5;
    const int k0w = (int)t.row0 + wid * 32, key = k0w + i;
    const bool live = key < t.lk;
    const int ahead = t.lk - t.lq;                             // causal: query x sees keys 0 .. x + ahead
    const float sl2 = p.scale * LOG2E;
    RowOperand<D> k, v;
    k.load(p.k + (t.k0 + (live ? key : 0)) * p.k_ss + w.head * p.k_sh, h, live);
    v.load(p.v + (t.k0 + (live ? key : 0)) * p.v_ss + w.head * p.v_sh, h, live);
    f32x16 dk[NDB], dv[NDB];
#pragma unroll
    for (int db = 0; db < NDB; ++db) { dk[db] = zero16(); dv[db] = zero16(); }
    // query tiles: from the first one that sees a key of this workgroup, for each of the g heads; this part's share of them
    const int first = p.causal ? max(0, (int)t.row0 - ahead) / KT * KT : 0;
    const int per_head = max(0, (t.lq - first + KT - 1) / KT);
    const long all = (long)per_head * p.g, per = (all + p.nsplit - 1) / p.nsplit;
    const int it0 = (int)min(all, w.part * per), it1 = (int)min(all, it0 + per);
    int hd = per_head > 0 ? it0 / per_head : 0, q0 = first + (it0 - hd * per_head) * KT;
    Staged<D> qs, ds;
    float st = 0.f;                                            // (rows past the sequence: zeros -- P = 1, but Q = dO = 0 and dS = 0)
    auto load = [&]() {
        const long head = (long)w.head * p.g + hd;
        const int x = q0 + threadIdx.x % KT;
        qs.load(p.q + t.q0 * p.q_ss + head * p.q_sh, p.q_ss, q0, t.lq);
        ds.load(p.dout + t.q0 * p.do_ss + head * p.do_sh, p.do_ss, q0, t.lq);
        if (threadIdx.x < 2 * KT) st = x < t.lq ? (threadIdx.x < KT ? p.lse : p.delta)[head * p.tq + t.q0 + x] : 0.f;
    };
    if (it0 < it1) load();
    for (int it = it0; it < it1; ++it) {
        __syncthreads();
        qs.store(Ql); ds.store(DOl);
        if (threadIdx.x < 2 * KT) stat[threadIdx.x / KT][threadIdx.x % KT] = st;
        __syncthreads();
        const int qt = q0;
        q0 += KT;
        if (q0 >= t.lq) { q0 = first; ++hd; }
        if (it + 1 < it1) load();
        if (k0w >= t.lk || (p.causal && qt + KT - 1 + ahead < k0w)) continue;      // wave-uniform: no live key, or none that a query of the tile sees
        f32x16 s = over_channels<D>(Ql, k, lane);
        const f32x16 dp = over_channels<D>(DOl, v, lane);
        f32x16 pr;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int x = entry_row(e, h);
            pr[e] = !p.causal || key <= qt + x + ahead ? __builtin_amdgcn_exp2f(s[e] * sl2 - stat[0][x]) : 0.f;
            s[e] = pr[e] * (dp[e] - stat[1][x]);
        }
        over_rows<D>(dv, DOl, pr, lane);
        over_rows<D>(dk, Ql, s, lane);
    }
    if (!live) return;
    const long row = ((t.k0 + key) * p.hk + w.head) * D, slice = p.tk * p.hk * D;
#pragma unroll
    for (int db = 0; db < NDB; ++db) {
        store_row((p.nsplit == 1 ? p.dk : p.part + 2 * w.part * slice) + row + 32 * db, dk[db], p.scale, h);
        store_row((p.nsplit == 1 ? p.dv : p.part + (2 * w.part + 1) * slice) + row + 32 * db, dv[db], 1.f, h);
    }
}

template <int D> void forward(const Params& p, hipStream_t s) {
    const unsigned grid = (unsigned)work_groups(row_slots(p.tq, p.g, p.n, ROWS), p.hk, p.nsplit);
    if (p.nsplit == 1) { varlen_f32_fwd_kernel<D, false><<<grid, NT, 0, s>>>(p); return; }
    varlen_f32_fwd_kernel<D, true><<<grid, NT, 0, s>>>(p);
    join<float, D>(p, s);
}
template <int D> void backward(const Params& p, hipStream_t s) {
    const unsigned rows = (unsigned)work_groups(row_slots(p.tq, p.g, p.n, ROWS), p.hk, p.dq_split);
    if (p.dq_split == 1) varlen_f32_dq_kernel<D, false><<<rows, NT, 0, s>>>(p);
    else { varlen_f32_dq_kernel<D, true><<<rows, NT, 0, s>>>(p); sum_parts(p, p.dq, (float*)nullptr, p.dq_split, p.tq * p.hq * D, s); }
    varlen_f32_dkv_kernel<D><<<(unsigned)work_groups(row_slots(p.tk, 1, p.n, ROWS), p.hk, p.nsplit), NT, 0, s>>>(p);
    if (p.nsplit > 1) sum_parts(p, p.dk, p.dv, p.nsplit, p.tk * p.hk * D, s);
}

}  // namespace

namespace dpipe_varlen {
void forward_f32(const VarlenParams<float>& p, int D, hipStream_t s) { if (D == 64) forward<64>(p, s); else forward<128>(p, s); }
void backward_f32(const VarlenParams<float>& p, int D, hipStream_t s) { if (D == 64) backward<64>(p, s); else backward<128>(p, s); }
}  // namespace dpipe_varlen
