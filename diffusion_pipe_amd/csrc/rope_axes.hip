// rope_axes.hip -- rotary positions with several axes (time, height, width; or one axis of text) on query and key heads, with their per-head RMS
// norms, forward + backward; bf16 or fp32 tensors, angles from the positions themselves (no cos / sin tables in memory).
//
//   n = x * rsqrt(mean(x^2) + eps) * w        (optional, per head row of D channels)
//   channel pair p of axis a:  theta = position[token][a] * f_p        (y0, y1) = (n0 cos - n1 sin, n1 cos + n0 sin)
//   backward:  g = R(-theta) gy;   dw = sum over tokens and heads of g * xhat;   u = g * w;   dx = r (u - xhat mean(u xhat)),  r = rsqrt(..), xhat = x r
//
// f_p comes from the host in fp64, in TURNS per unit of position; the turn count position * f_p and its reduction to one turn are fp64 as well (a position
// of 10^6 keeps 10 digits of its angle), sine and cosine of the remainder fp32.  Pairs are neighbours (2 p, 2 p + 1) or halves (p, p + R / 2) of the R
// rotated channels; channels behind R pass through (normalised, not rotated).
//
// Bound: HBM (forward reads x and writes y once, the backward of a normed row reads x and gy and writes dx).  61 456 tokens x (24 + 24) heads of 128 in bf16 with norms: forward
// 1.51 GB in 256 us = 5.9 TB/s, backward 2.27 GB in 400 us = 5.7 TB/s (a copy of 2 GiB: 4.8); 4608 tokens of the same heads, cached: 22 us.
// One workgroup takes up to 8 tokens: its threads make the tokens' (cos, sin) pairs in LDS once, then every head row of q and of k uses them -- the trigonometry (fp64 turns) is
// paid once per token, not per head, and no table is read.  A head row is LPR lanes of 8 channels; the norm's sums stay inside the lane group, by operand modifiers of the add
// instead of LDS exchanges, and 4 rows a lane group are in flight (forward 286 -> 272 us, then 258 with streaming accesses).
#include <cstdio>
#include "dpipe_common.h"
#include "../../include/dpipe_hip.h"

using namespace dpipe;

namespace {

constexpr int NB = 256;
constexpr int MAX_PAIRS = 128;           // head dim <= 256
constexpr int TABLE = 256;               // (cos, sin) pairs in LDS: tokens of a tile * pairs (rounded up to 4) <= TABLE
constexpr int AHEAD = 4;                 // rows of a lane group that are in flight
constexpr int MAX_BWD_BLOCKS = 512;      // partial rows of a weight's gradient: with both tensors 4 workgroups per CU

struct RopeAxesParams {
    const void *x[2], *gy[2], *w[2];     // [0] query, [1] key
    void* y[2];
    const void* pos;
    float* part;                         // weight gradient partials [blocks][2][D]
    long x_ss[2], x_sh[2], g_ss[2], g_sh[2];
    long tokens, period;                 // positions repeat every `period` tokens
    int heads[2];
    int D, pairs, axes, tb, pos_type, w_f32[2];
    int stream;                          // the tensors are larger than the last-level cache
    unsigned pair_magic;                 // ceil(2^32 / pairs): entry / pairs of a table by multiplication
    int step_t[2], step_h[2];            // lane groups per workgroup = step_t heads + step_h: a lane group's next row is step_t tokens and step_h heads further
    float eps, sign;                     // sign = -1: the inverse rotation
    double freq[MAX_PAIRS];
    unsigned char axis[MAX_PAIRS];
};

template <typename T> __device__ __forceinline__ void load4(const T* p, float* f);
template <> __device__ __forceinline__ void load4<bf16_t>(const bf16_t* p, float* f) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    f[0] = __uint_as_float(u.x << 16); f[1] = __uint_as_float(u.x & 0xffff0000u); f[2] = __uint_as_float(u.y << 16); f[3] = __uint_as_float(u.y & 0xffff0000u);
}
template <> __device__ __forceinline__ void load4<float>(const float* p, float* f) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    f[0] = u.x; f[1] = u.y; f[2] = u.z; f[3] = u.w;
}

// the 8 channels of a lane as loaded, 16 (bf16) or 32 (fp32) bytes: neighbours pairing = channels 8 l .. 8 l + 7, halves pairing = 4 channels of either half
// STREAM: past the caches (tensors that no cache holds until they are read again)
template <bool STREAM, typename V> __device__ __forceinline__ V get_vec(const void* p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p)); else return *reinterpret_cast<const V*>(p);
}
template <bool STREAM, typename V> __device__ __forceinline__ void put_vec(void* p, V v) {
    if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<V*>(p)); else *reinterpret_cast<V*>(p) = v;
}
typedef __attribute__((ext_vector_type(2))) unsigned int u32x2_t;

template <typename T, bool HALF, bool STREAM> struct Raw8 {
    u32x4_t v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p, int c0, int c1) {
        if constexpr (sizeof(T) == 4) {
            v[0] = get_vec<STREAM, u32x4_t>(p + c0); v[1] = get_vec<STREAM, u32x4_t>(p + c1);
        } else if constexpr (HALF) {
            const u32x2_t a = get_vec<STREAM, u32x2_t>(p + c0), b = get_vec<STREAM, u32x2_t>(p + c1);
            v[0] = u32x4_t{a.x, a.y, b.x, b.y};
        } else {
            v[0] = get_vec<STREAM, u32x4_t>(p + c0);
        }
    }
    __device__ __forceinline__ void store(T* p, int c0, int c1) const {
        if constexpr (sizeof(T) == 4) {
            put_vec<STREAM>(p + c0, v[0]); put_vec<STREAM>(p + c1, v[1]);
        } else if constexpr (HALF) {
            put_vec<STREAM>(p + c0, u32x2_t{v[0].x, v[0].y}); put_vec<STREAM>(p + c1, u32x2_t{v[0].z, v[0].w});
        } else {
            put_vec<STREAM>(p + c0, v[0]);
        }
    }
    __device__ __forceinline__ void unpack(float* f) const {
        Vec16<T> u;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) { u.raw = __builtin_bit_cast(uint4, v[i]); u.unpack(f + i * Vec16<T>::N); }
    }
    __device__ __forceinline__ void pack(const float* f) {
        Vec16<T> u;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) { u.pack(f + i * Vec16<T>::N); v[i] = __builtin_bit_cast(u32x4_t, u.raw); }
    }
};

// sum over groups of LPR lanes, in every lane: exchanges inside 16 lanes are operand modifiers of the add (no LDS)
template <int CTRL> __device__ __forceinline__ float add_dpp(float v) { return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)); }
template <int LPR> __device__ __forceinline__ float group_sum(float v) {
    v = add_dpp<0xb1>(v);                                    // lane ^ 1
    v = add_dpp<0x4e>(v);                                    // lane ^ 2
    v = add_dpp<0x141>(v);                                   // mirrored in 8: the other four
    if (LPR > 8) v = add_dpp<0x140>(v);                      // mirrored in 16: the other eight
    if (LPR > 16) v += __shfl_xor(v, 16, 64);
    return v;
}

__device__ __forceinline__ double position(const RopeAxesParams& p, long token, int axis) {
    const long i = (token < p.period ? token : token % p.period) * p.axes + axis;
    if (p.pos_type == 2) return (double)reinterpret_cast<const long long*>(p.pos)[i];
    if (p.pos_type == 1) return (double)reinterpret_cast<const int*>(p.pos)[i];
    return (double)reinterpret_cast<const float*>(p.pos)[i];
}

// (cos, sin) of the tile's tokens into LDS, `pitch` entries a token; `sign` turns the rotation round
__device__ __forceinline__ int table_pitch(int pairs) { return (pairs + 3) & ~3; }
__device__ __forceinline__ void fill_table(const RopeAxesParams& p, float* table, long t0, int ntok) {
    for (int e = threadIdx.x; e < ntok * p.pairs; e += NB) {
        const int t = p.pairs == 1 ? e : (int)__umulhi((unsigned)e, p.pair_magic), pr = e - t * p.pairs;
        double turns = position(p, t0 + t, p.axis[pr]) * p.freq[pr];
        turns -= rint(turns);
        float s, c;
        sincospif(2.f * (float)turns, &s, &c);
        table[t * table_pitch(p.pairs) + pr] = c;
        table[TABLE + t * table_pitch(p.pairs) + pr] = p.sign * s;
    }
}

// the lane's four pairs, from p0 on, of one token: channels (2 j, 2 j + 1) of its 8, or (j, 4 + j) with halves pairing.  Pairs behind the rotated ones keep their bits.
template <bool HALF> __device__ __forceinline__ void rotate(float* f, const float* table, int p0, int pairs, bool full) {
    const float4 vc = *reinterpret_cast<const float4*>(table + p0), vs = *reinterpret_cast<const float4*>(table + TABLE + p0);
    const float c[4] = {vc.x, vc.y, vc.z, vc.w}, s[4] = {vs.x, vs.y, vs.z, vs.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int a = HALF ? j : 2 * j, b = HALF ? 4 + j : 2 * j + 1;
        const float y0 = f[a] * c[j] - f[b] * s[j], y1 = f[b] * c[j] + f[a] * s[j];
        const bool rot = full || p0 + j < pairs;
        f[a] = rot ? y0 : f[a]; f[b] = rot ? y1 : f[b];
    }
}

template <bool HALF> __device__ __forceinline__ void lane_channels(const RopeAxesParams& p, int sub, int& c0, int& c1) {
    c0 = 8 * sub; c1 = c0 + 4;
    if (HALF && 4 * sub < p.pairs) { c0 = 4 * sub; c1 = p.pairs + 4 * sub; }
}

__device__ __forceinline__ void load_weight(const RopeAxesParams& p, int which, int c0, int c1, float* w) {
    if (p.w_f32[which]) { load4(reinterpret_cast<const float*>(p.w[which]) + c0, w); load4(reinterpret_cast<const float*>(p.w[which]) + c1, w + 4); }
    else { load4(reinterpret_cast<const bf16_t*>(p.w[which]) + c0, w); load4(reinterpret_cast<const bf16_t*>(p.w[which]) + c1, w + 4); }
}

// A lane group's walk over the head rows of a tile (row = token * heads + head, one row every GROUPS): offsets inside the tile fit 32 bits (the launcher sees to it)
struct Walk {
    int token, head;
    __device__ __forceinline__ void start(int grp, int heads) { token = grp / heads; head = grp - token * heads; }
    __device__ __forceinline__ void next(int step_t, int step_h, int heads) {
        token += step_t; head += step_h;
        const bool over = head >= heads;
        token += over ? 1 : 0; head -= over ? heads : 0;
    }
    __device__ __forceinline__ unsigned offset(int ss, int sh) const { return (unsigned)(token * ss + head * sh); }
};

// What a lane keeps of its place in the workgroup
template <bool HALF, int LPR> struct Lane {
    int sub, grp, c0 = 0, c1 = 4, p0;
    bool in, full;
    __device__ __forceinline__ Lane(const RopeAxesParams& p) {
        sub = threadIdx.x % LPR; grp = threadIdx.x / LPR;
        in = 8 * sub < p.D; full = 2 * p.pairs == p.D;
        if (in) lane_channels<HALF>(p, sub, c0, c1);
        p0 = 4 * sub < p.pairs ? 4 * sub : 0;                // (lanes behind the rotated channels read the table somewhere and keep their values)
    }
};

// The rows of one tensor of a tile: y = R [norm](x)
template <typename T, int LPR, bool HALF, bool STREAM, bool NORM>
__device__ __forceinline__ void rows_forward(const RopeAxesParams& p, const Lane<HALF, LPR>& ln, const float* table, int which, long t0, int ntok, Raw8<T, HALF, STREAM>* raw, bool loaded) {
    constexpr int GROUPS = NB / LPR;
    const int heads = p.heads[which], rows = ntok * heads, iters = (rows + GROUPS - 1) / GROUPS, pitch = table_pitch(p.pairs);
    const int ss = (int)p.x_ss[which], sh = (int)p.x_sh[which], st = p.step_t[which], sd = p.step_h[which];
    const T* x = reinterpret_cast<const T*>(p.x[which]) + t0 * p.x_ss[which];
    T* y = reinterpret_cast<T*>(p.y[which]) + t0 * heads * (long)p.D;
    const float inv_d = 1.f / (float)p.D;
    float w[8];
    if (NORM) load_weight(p, which, ln.c0, ln.c1, w);
    Walk get, put;
    get.start(ln.grp, heads); put.start(ln.grp, heads);
    auto fetch = [&](Raw8<T, HALF, STREAM>& r) {
        if (get.token < ntok) r.load(x + get.offset(ss, sh), ln.c0, ln.c1);
        get.next(st, sd, heads);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) fetch(raw[u]);
    if (!loaded) __syncthreads();                            // the table is complete
    for (int i = 0; i < iters; i += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (i + u >= iters) break;                       // (uniform)
            float f[8];
            raw[u].unpack(f);
            fetch(raw[u]);
            if (NORM) {
                float sq = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) sq += f[j] * f[j];
                const float rstd = rsqrtf(group_sum<LPR>(ln.in ? sq : 0.f) * inv_d + p.eps);
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = f[j] * rstd * w[j];
            }
            const bool live = ln.in && put.token < ntok;
            rotate<HALF>(f, table + (put.token < ntok ? put.token * pitch : 0), ln.p0, ln.in && 4 * ln.sub < p.pairs ? p.pairs : 0, ln.full);
            Raw8<T, HALF, STREAM> out;
            out.pack(f);
            if (live) out.store(y + (unsigned)((put.token * heads + put.head) * p.D), ln.c0, ln.c1);
            put.next(st, sd, heads);
        }
    }
}

// y = R(sign * theta) [norm](x): the forward, and the backward of rows without a norm (sign = -1)
template <typename T, int LPR, bool HALF, bool STREAM>
__global__ void __launch_bounds__(NB) rope_axes_kernel(const RopeAxesParams p) {
    __shared__ __attribute__((aligned(16))) float table[2 * TABLE];     // cosines, then sines
    const Lane<HALF, LPR> ln(p);
    const long t0 = (long)blockIdx.x * p.tb;
    const int ntok = (int)min((long)p.tb, p.tokens - t0);
    fill_table(p, table, t0, ntok);
    Raw8<T, HALF, STREAM> raw[AHEAD];
    if (p.w[0]) rows_forward<T, LPR, HALF, STREAM, true>(p, ln, table, 0, t0, ntok, raw, false); else rows_forward<T, LPR, HALF, STREAM, false>(p, ln, table, 0, t0, ntok, raw, false);
    if (p.heads[1] == 0) return;
    if (p.w[1]) rows_forward<T, LPR, HALF, STREAM, true>(p, ln, table, 1, t0, ntok, raw, true); else rows_forward<T, LPR, HALF, STREAM, false>(p, ln, table, 1, t0, ntok, raw, true);
}

// The backward of one tensor's rows of a tile: dx, and the weight's gradient added to the lane's dw
template <typename T, int LPR, bool HALF, bool STREAM, bool NORM>
__device__ __forceinline__ void rows_backward(const RopeAxesParams& p, const Lane<HALF, LPR>& ln, const float* table, int which, long t0, int ntok, const float* w, float* dw) {
    constexpr int GROUPS = NB / LPR, A = 2;
    const int heads = p.heads[which], rows = ntok * heads, iters = (rows + GROUPS - 1) / GROUPS, pitch = table_pitch(p.pairs);
    const int ss = (int)p.x_ss[which], sh = (int)p.x_sh[which], gs = (int)p.g_ss[which], gh = (int)p.g_sh[which], st = p.step_t[which], sd = p.step_h[which];
    const T* x = reinterpret_cast<const T*>(p.x[which]) + t0 * p.x_ss[which];
    const T* gy = reinterpret_cast<const T*>(p.gy[which]) + t0 * p.g_ss[which];
    T* dx = reinterpret_cast<T*>(p.y[which]) + t0 * heads * (long)p.D;
    const float inv_d = 1.f / (float)p.D;
    Raw8<T, HALF, STREAM> rx[A], rg[A];
    Walk get, put;
    get.start(ln.grp, heads); put.start(ln.grp, heads);
    auto fetch = [&](int u) {
        if (get.token < ntok) {
            if (NORM) rx[u].load(x + get.offset(ss, sh), ln.c0, ln.c1);
            rg[u].load(gy + get.offset(gs, gh), ln.c0, ln.c1);
        }
        get.next(st, sd, heads);
    };
#pragma unroll
    for (int u = 0; u < A; ++u) fetch(u);
    __syncthreads();                                         // the table is complete
    for (int i = 0; i < iters; i += A) {
#pragma unroll
        for (int u = 0; u < A; ++u) {
            if (i + u >= iters) break;
            float f[8], g[8];
            rg[u].unpack(g);
            if (NORM) rx[u].unpack(f);
            fetch(u);
            const bool live = ln.in && put.token < ntok;
            rotate<HALF>(g, table + (put.token < ntok ? put.token * pitch : 0), ln.p0, ln.in && 4 * ln.sub < p.pairs ? p.pairs : 0, ln.full);
            if (NORM) {
                float sq = 0.f, dot = 0.f;                   // sum x^2 and sum u x:  mean(u xhat) = r * dot / D
#pragma unroll
                for (int j = 0; j < 8; ++j) { sq += f[j] * f[j]; dot += g[j] * w[j] * f[j]; }
                sq = group_sum<LPR>(ln.in ? sq : 0.f); dot = group_sum<LPR>(ln.in ? dot : 0.f);
                const float rstd = rsqrtf(sq * inv_d + p.eps), m = rstd * dot * inv_d;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float xh = f[j] * rstd;
                    dw[j] += live ? g[j] * xh : 0.f;
                    g[j] = rstd * (g[j] * w[j] - xh * m);
                }
            }
            Raw8<T, HALF, STREAM> out;
            out.pack(g);
            if (live) out.store(dx + (unsigned)((put.token * heads + put.head) * p.D), ln.c0, ln.c1);
            put.next(st, sd, heads);
        }
    }
}

// the backward with norms: dx, and per workgroup one partial row of the weight's gradient (summed in a fixed order by rope_axes_dw_kernel).  A workgroup takes the tiles of one
// tensor (blockIdx.y): with both, the weights and their gradients of both sit in registers and 4 waves a SIMD spill.
template <typename T, int LPR, bool HALF, bool STREAM>
__global__ void __launch_bounds__(NB, 4) rope_axes_bwd_kernel(const RopeAxesParams p) {
    constexpr int GROUPS = NB / LPR;
    __shared__ __attribute__((aligned(16))) float table[2 * TABLE];     // cosines, then sines
    __shared__ float red[GROUPS][LPR * 8];
    const Lane<HALF, LPR> ln(p);
    const int which = blockIdx.y;
    const bool norm = p.w[which] != nullptr;
    float w[8], dw[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) { w[j] = 1.f; dw[j] = 0.f; }
    if (norm) load_weight(p, which, ln.c0, ln.c1, w);
    for (long t0 = (long)blockIdx.x * p.tb; t0 < p.tokens; t0 += (long)gridDim.x * p.tb) {
        const int ntok = (int)min((long)p.tb, p.tokens - t0);
        __syncthreads();                                       // the previous tile's rows are done with the table
        fill_table(p, table, t0, ntok);
        if (norm) rows_backward<T, LPR, HALF, STREAM, true>(p, ln, table, which, t0, ntok, w, dw);
        else rows_backward<T, LPR, HALF, STREAM, false>(p, ln, table, which, t0, ntok, w, dw);
    }
    __syncthreads();
    if (ln.in) {
#pragma unroll
        for (int j = 0; j < 4; ++j) { red[ln.grp][ln.c0 + j] = dw[j]; red[ln.grp][ln.c1 + j] = dw[4 + j]; }
    }
    __syncthreads();
    if ((int)threadIdx.x < p.D) {
        float s = 0.f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) s += red[g][threadIdx.x];
        p.part[((long)blockIdx.x * 2 + which) * p.D + threadIdx.x] = s;
    }
}

// dw[c] (+)= sum over `blocks` partial rows, in a fixed order: 32 columns (8 lanes of 4) x 32 slices of the rows per workgroup.  Latency: 5.6 us for 512 rows.
__global__ void __launch_bounds__(NB) rope_axes_dw_kernel(const float* __restrict__ part, void* dq, void* dk, int q_f32, int k_f32, int accumulate_q, int accumulate_k,
                                                          int blocks, int D) {
    __shared__ __attribute__((aligned(16))) float red[32][32];
    const int ct = 4 * (threadIdx.x & 7), sl = threadIdx.x >> 3, which = blockIdx.y, c = blockIdx.x * 32 + ct;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (c < D) {
#pragma unroll 16
        for (int s = sl; s < blocks; s += 32) {
            const float4 v = *reinterpret_cast<const float4*>(part + ((long)s * 2 + which) * D + c);
            a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
        }
    }
    *reinterpret_cast<float4*>(&red[sl][ct]) = a;
    __syncthreads();
    void* out = which ? dk : dq;
    const int col = blockIdx.x * 32 + threadIdx.x;
    if (threadIdx.x < 32 && col < D && out) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) s += red[r][threadIdx.x];
        const bool f32 = which ? k_f32 : q_f32, acc = which ? accumulate_k : accumulate_q;
        if (f32) { float* o = reinterpret_cast<float*>(out) + col; *o = acc ? *o + s : s; }
        else { bf16_t* o = reinterpret_cast<bf16_t*>(out) + col; *o = f32_to_bf16(acc ? bf16_to_f32(*o) + s : s); }
    }
}

// tokens per workgroup: as many as the table holds, while 1 024 workgroups (4 per CU) are left
int tile_tokens(long tokens, int pairs) {
    int tb = TABLE / ((pairs + 3) & ~3);
    if (tb > 8) tb = 8;
    while (tb > 1 && (tokens + tb - 1) / tb < 1024) --tb;
    return tb;
}

// 8 tokens and all heads stay within 2^29 elements of the tile's first (32-bit byte offsets)
bool rows_fit(long ss, long sh, int heads) { return ss >= 0 && sh >= 0 && ss < (1l << 25) && sh * heads < (1l << 28); }
bool rows_ok(const void* p, long ss, long sh) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ss % 8 == 0 && sh % 8 == 0; }

int lanes_per_row(int D) { return D <= 64 ? 8 : D <= 128 ? 16 : 32; }

// checks shared by both entry points; fills everything but the gradient operands
int fill(RopeAxesParams& p, const char* what, const void* q, const void* k, const void* pos, int pos_type, const double* freq, const int* axis, long tokens, long period,
         int axes, int pairs, int heads_q, int heads_k, int D, long q_ss, long q_sh, long k_ss, long k_sh, const void* wq, const void* wk, int wq_dt, int wk_dt, float eps,
         int half, int dt) {
    auto bad = [&](const char* m) { static thread_local char buf[160]; snprintf(buf, sizeof(buf), "%s: %s", what, m); set_last_error(buf); return DPIPE_ERR_ARG; };
    if (!q || !pos || tokens <= 0 || period <= 0 || heads_q <= 0 || heads_k < 0 || (heads_k > 0 && !k) || axes <= 0) return bad("bad argument");
    if (dt != DPIPE_BF16 && dt != DPIPE_F32) return bad("dtype must be bf16 or fp32");
    if (D <= 0 || D > 256 || D % 8) return bad("head dim must be a multiple of 8 up to 256");
    if (pairs <= 0 || 2 * pairs > D || (half && pairs % 4)) return bad("rotated channels must fit the head (halves pairing: a multiple of 8)");
    if (!freq || !axis || heads_q > 4096 || heads_k > 4096) return bad("bad argument");
    if (pos_type < 0 || pos_type > 2) return bad("positions must be fp32, int32 or int64");
    if (!rows_ok(q, q_ss, q_sh) || (heads_k > 0 && !rows_ok(k, k_ss, k_sh)) || (reinterpret_cast<uintptr_t>(wq) & 15) || (reinterpret_cast<uintptr_t>(wk) & 15))
        return bad("tensors must be 16-byte aligned with strides multiple of 8 elements");
    if (!rows_fit(q_ss, q_sh, heads_q) || (heads_k > 0 && !rows_fit(k_ss, k_sh, heads_k))) return bad("strides too large");
    if ((wq && wq_dt != DPIPE_BF16 && wq_dt != DPIPE_F32) || (wk && wk_dt != DPIPE_BF16 && wk_dt != DPIPE_F32)) return bad("weights must be bf16 or fp32");
    p.x[0] = q; p.x[1] = k; p.x_ss[0] = q_ss; p.x_sh[0] = q_sh; p.x_ss[1] = k_ss; p.x_sh[1] = k_sh;
    p.pos = pos; p.pos_type = pos_type; p.tokens = tokens; p.period = period; p.axes = axes; p.pairs = pairs; p.D = D;
    p.heads[0] = heads_q; p.heads[1] = heads_k; p.w[0] = wq; p.w[1] = heads_k > 0 ? wk : nullptr;
    p.w_f32[0] = wq_dt == DPIPE_F32; p.w_f32[1] = wk_dt == DPIPE_F32; p.eps = eps;
    // 256 MB of last-level cache: below, what is written here is read from it by the attention that follows, and the forward's rows by the backward; above, streaming past it is faster
    // (755 MB of heads: forward 271 -> 255 us = 5.9 TB/s, backward 443 -> 413; 57 MB: 21.3 us cached, 22.6 streamed)
    p.stream = tokens * (long)(heads_q + heads_k) * D * (dt == DPIPE_F32 ? 4 : 2) > (256l << 20);
    p.pair_magic = (unsigned)((0x100000000ull + pairs - 1) / pairs);
    const int groups = NB / lanes_per_row(D);
    for (int w = 0; w < 2; ++w) { const int h = p.heads[w] > 0 ? p.heads[w] : 1; p.step_t[w] = groups / h; p.step_h[w] = groups % h; }
    for (int i = 0; i < pairs; ++i) {
        if (axis[i] < 0 || axis[i] >= axes || axis[i] > 255) return bad("axis index out of range (below axes and 256)");
        p.freq[i] = freq[i]; p.axis[i] = (unsigned char)axis[i];
    }
    p.tb = tile_tokens(tokens, pairs);
    if (cdiv(tokens, p.tb) >= (1l << 23)) return bad("too many tokens");
    return DPIPE_OK;
}

template <typename T, bool HALF, bool STREAM> void launch(const RopeAxesParams& p, bool backward, unsigned blocks, hipStream_t s) {
    const dim3 grid(blocks, backward && p.heads[1] > 0 ? 2 : 1);
#define LAUNCH(LPR) do { if (backward) rope_axes_bwd_kernel<T, LPR, HALF, STREAM><<<grid, NB, 0, s>>>(p); else rope_axes_kernel<T, LPR, HALF, STREAM><<<grid, NB, 0, s>>>(p); } while (0)
    switch (lanes_per_row(p.D)) { case 8: LAUNCH(8); break; case 16: LAUNCH(16); break; default: LAUNCH(32); }
#undef LAUNCH
}
// backward: the kernel with norms (without, the backward is the forward's kernel with the sign turned round)
void launch(const RopeAxesParams& p, int dtype, bool half, bool backward, unsigned blocks, hipStream_t s) {
    auto with = [&](auto type) {
        typedef decltype(type) T;
        if (half) { if (p.stream) launch<T, true, true>(p, backward, blocks, s); else launch<T, true, false>(p, backward, blocks, s); }
        else { if (p.stream) launch<T, false, true>(p, backward, blocks, s); else launch<T, false, false>(p, backward, blocks, s); }
    };
    if (dtype == DPIPE_BF16) with(bf16_t{}); else with(float{});
}

}  // namespace

extern "C" {

int dpipe_rope_axes_fwd(const void* q, const void* k, const void* positions, int pos_type, const double* freq, const int* axis, const void* wq, const void* wk, void* yq,
                        void* yk, long tokens, long period, int axes, int pairs, int heads_q, int heads_k, int D, long q_ss, long q_sh, long k_ss, long k_sh, float eps,
                        int half, int dtype, int wq_dtype, int wk_dtype, void* stream) {
    RopeAxesParams p = {};
    const int rc = fill(p, "dpipe_rope_axes_fwd", q, k, positions, pos_type, freq, axis, tokens, period, axes, pairs, heads_q, heads_k, D, q_ss, q_sh, k_ss, k_sh, wq, wk,
                        wq_dtype, wk_dtype, eps, half, dtype);
    if (rc) return rc;
    if (!yq || (heads_k > 0 && !yk) || !aligned16(yq) || !aligned16(yk)) { set_last_error("dpipe_rope_axes_fwd: bad output"); return DPIPE_ERR_ARG; }
    p.y[0] = yq; p.y[1] = yk; p.sign = 1.f;
    launch(p, dtype, half, false, (unsigned)cdiv(p.tokens, p.tb), reinterpret_cast<hipStream_t>(stream));
    return check_launch("dpipe_rope_axes_fwd");
}

long dpipe_rope_axes_workspace_floats(int D) { return 2l * MAX_BWD_BLOCKS * D; }

int dpipe_rope_axes_bwd(const void* q, const void* k, const void* gq, const void* gk, const void* positions, int pos_type, const double* freq, const int* axis, const void* wq,
                        const void* wk, void* dq, void* dk, void* dwq, void* dwk, float* ws, long tokens, long period, int axes, int pairs, int heads_q, int heads_k, int D,
                        long q_ss, long q_sh, long k_ss, long k_sh, long gq_ss, long gq_sh, long gk_ss, long gk_sh, float eps, int half, int dtype, int wq_dtype, int wk_dtype,
                        int accumulate_wq, int accumulate_wk, void* stream) {
    RopeAxesParams p = {};
    const int rc = fill(p, "dpipe_rope_axes_bwd", q, k, positions, pos_type, freq, axis, tokens, period, axes, pairs, heads_q, heads_k, D, q_ss, q_sh, k_ss, k_sh, wq, wk,
                        wq_dtype, wk_dtype, eps, half, dtype);
    if (rc) return rc;
    if (!gq || (heads_k > 0 && !gk) || !rows_ok(gq, gq_ss, gq_sh) || !rows_fit(gq_ss, gq_sh, heads_q) ||
        (heads_k > 0 && (!rows_ok(gk, gk_ss, gk_sh) || !rows_fit(gk_ss, gk_sh, heads_k))) || !dq || (heads_k > 0 && !dk) || !aligned16(dq) || !aligned16(dk)) {
        set_last_error("dpipe_rope_axes_bwd: gradients must be 16-byte aligned with strides multiple of 8 elements, not too large"); return DPIPE_ERR_ARG; }
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    p.y[0] = dq; p.y[1] = dk; p.sign = -1.f;
    if (!p.w[0] && !p.w[1]) {                                  // no norm: the inverse rotation of the gradient
        p.x[0] = gq; p.x[1] = gk; p.x_ss[0] = gq_ss; p.x_sh[0] = gq_sh; p.x_ss[1] = gk_ss; p.x_sh[1] = gk_sh;
        launch(p, dtype, half, false, (unsigned)cdiv(p.tokens, p.tb), s);
        return check_launch("dpipe_rope_axes_bwd");
    }
    if (!ws) { set_last_error("dpipe_rope_axes_bwd: a normed row needs the workspace"); return DPIPE_ERR_ARG; }
    p.gy[0] = gq; p.gy[1] = gk; p.g_ss[0] = gq_ss; p.g_sh[0] = gq_sh; p.g_ss[1] = gk_ss; p.g_sh[1] = gk_sh; p.part = ws;
    const long tiles = cdiv(tokens, p.tb);
    const unsigned grid = (unsigned)(tiles < MAX_BWD_BLOCKS ? tiles : MAX_BWD_BLOCKS);
    launch(p, dtype, half, true, grid, s);
    if (dwq || dwk)
        rope_axes_dw_kernel<<<dim3((unsigned)cdiv(D, 32), 2), NB, 0, s>>>(ws, dwq, dwk, wq_dtype == DPIPE_F32, wk_dtype == DPIPE_F32, accumulate_wq, accumulate_wk, (int)grid, D);
    return check_launch("dpipe_rope_axes_bwd");
}

}  // extern "C"
