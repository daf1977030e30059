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
// Bound: HBM (forward reads x and writes y once, the backward of a normed row reads x and gy and writes dx).  One workgroup takes TB tokens: its threads
// make the TB * R / 2 (cos, sin) pairs in LDS once, then every head row of q and of k uses them -- the trigonometry is paid once per token, not
// per head.  A head row is LPR lanes of 8 channels; the norm's sums stay inside the lane group.
#include <cstdio>
#include "dpipe_common.h"
#include "../../include/dpipe_hip.h"

using namespace dpipe;

namespace {

constexpr int NB = 256;
constexpr int MAX_PAIRS = 128;           // head dim <= 256
constexpr int TABLE = 256;               // (cos, sin) pairs in LDS: TB * pairs <= TABLE
constexpr int MAX_BWD_BLOCKS = 1024;     // partial rows of the weight gradient: 4 workgroups per CU

struct RopeAxesParams {
    const void *x[2], *gy[2], *w[2];     // [0] query, [1] key
    void* y[2];
    const void* pos;
    float* part;                         // weight gradient partials [blocks][2][D]
    long x_ss[2], x_sh[2], g_ss[2], g_sh[2];
    long tokens, period;                 // positions repeat every `period` tokens
    int heads[2];
    int D, pairs, axes, tb, pos_type, w_f32[2];
    unsigned magic[2];                   // ceil(2^32 / heads): row / heads for rows < 2^16
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
template <typename T, bool HALF> struct Raw8 {
    uint4 v[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p, int c0, int c1) {
        if constexpr (sizeof(T) == 4) {
            v[0] = *reinterpret_cast<const uint4*>(p + c0); v[1] = *reinterpret_cast<const uint4*>(p + c1);
        } else if constexpr (HALF) {
            const uint2 a = *reinterpret_cast<const uint2*>(p + c0), b = *reinterpret_cast<const uint2*>(p + c1);
            v[0] = make_uint4(a.x, a.y, b.x, b.y);
        } else {
            v[0] = *reinterpret_cast<const uint4*>(p + c0);
        }
    }
    __device__ __forceinline__ void store(T* p, int c0, int c1) const {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<uint4*>(p + c0) = v[0]; *reinterpret_cast<uint4*>(p + c1) = v[1];
        } else if constexpr (HALF) {
            *reinterpret_cast<uint2*>(p + c0) = make_uint2(v[0].x, v[0].y); *reinterpret_cast<uint2*>(p + c1) = make_uint2(v[0].z, v[0].w);
        } else {
            *reinterpret_cast<uint4*>(p + c0) = v[0];
        }
    }
    __device__ __forceinline__ void unpack(float* f) const {
        Vec16<T> u;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) { u.raw = v[i]; u.unpack(f + i * Vec16<T>::N); }
    }
    __device__ __forceinline__ void pack(const float* f) {
        Vec16<T> u;
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) { u.pack(f + i * Vec16<T>::N); v[i] = u.raw; }
    }
};

template <int LPR> __device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ double position(const RopeAxesParams& p, long token, int axis) {
    const long i = (token % p.period) * p.axes + axis;
    if (p.pos_type == 2) return (double)reinterpret_cast<const long long*>(p.pos)[i];
    if (p.pos_type == 1) return (double)reinterpret_cast<const int*>(p.pos)[i];
    return (double)reinterpret_cast<const float*>(p.pos)[i];
}

// (cos, sin) of the tile's tokens into LDS; `sign` turns the rotation round
__device__ __forceinline__ void fill_table(const RopeAxesParams& p, float2* table, long t0, int ntok) {
    for (int e = threadIdx.x; e < ntok * p.pairs; e += NB) {
        const int t = e / p.pairs, pr = e - t * p.pairs;
        double turns = position(p, t0 + t, p.axis[pr]) * p.freq[pr];
        turns -= rint(turns);
        float s, c;
        sincospif(2.f * (float)turns, &s, &c);
        table[e] = make_float2(c, p.sign * s);
    }
}

// pair j of the lane: f[.] rotated in place where `rot`; PAIR j = channels (2 j, 2 j + 1) of the lane's 8, or (j, 4 + j) with halves pairing
template <bool HALF> __device__ __forceinline__ void rotate(float* f, const float2* cs, int p0, int pairs) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int a = HALF ? j : 2 * j, b = HALF ? 4 + j : 2 * j + 1;
        const bool rot = p0 + j < pairs;
        const float2 t = cs[rot ? p0 + j : 0];
        const float y0 = f[a] * t.x - f[b] * t.y, y1 = f[b] * t.x + f[a] * t.y;
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

// y = R(sign * theta) [norm](x): the forward, and the backward of rows without a norm (sign = -1)
template <typename T, int LPR, bool HALF, bool NORM>
__global__ void __launch_bounds__(NB) rope_axes_kernel(const RopeAxesParams p) {
    constexpr int GROUPS = NB / LPR, U = 4;                   // U rows of a lane group in flight
    __shared__ float2 table[TABLE];
    const int sub = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const long t0 = (long)blockIdx.x * p.tb;
    const int ntok = (int)min((long)p.tb, p.tokens - t0);
    fill_table(p, table, t0, ntok);
    __syncthreads();
    const bool in = 8 * sub < p.D;
    int c0 = 0, c1 = 4;
    if (in) lane_channels<HALF>(p, sub, c0, c1);
    const float inv_d = 1.f / (float)p.D;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        const int heads = p.heads[which];
        const bool norm = NORM && p.w[which] != nullptr;
        float w[8];
        if (norm) load_weight(p, which, c0, c1, w);
        const T* x = reinterpret_cast<const T*>(p.x[which]) + t0 * p.x_ss[which];
        T* y = reinterpret_cast<T*>(p.y[which]) + t0 * heads * (long)p.D;
        const int rows = ntok * heads;
        for (int r0 = grp; r0 < rows; r0 += GROUPS * U) {
            Raw8<T, HALF> raw[U];
            int tl[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = min(r0 + u * GROUPS, rows - 1);
                tl[u] = heads == 1 ? r : (int)__umulhi((unsigned)r, p.magic[which]);
                raw[u].load(x + tl[u] * p.x_ss[which] + (r - tl[u] * heads) * p.x_sh[which], c0, c1);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + u * GROUPS;
                float f[8];
                raw[u].unpack(f);
                if (norm) {
                    float ss = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
                    const float rstd = rsqrtf(group_sum<LPR>(in ? ss : 0.f) * inv_d + p.eps);
#pragma unroll
                    for (int j = 0; j < 8; ++j) f[j] = f[j] * rstd * w[j];
                }
                rotate<HALF>(f, table + tl[u] * p.pairs, 4 * sub, p.pairs);
                raw[u].pack(f);
                if (in && r < rows) raw[u].store(y + (long)r * p.D, c0, c1);
            }
        }
    }
}

// the backward with norms: dx, and per workgroup one partial row of either weight's gradient (summed in a fixed order by rope_axes_dw_kernel)
template <typename T, int LPR, bool HALF>
__global__ void __launch_bounds__(NB) rope_axes_bwd_kernel(const RopeAxesParams p) {
    constexpr int GROUPS = NB / LPR, U = 2;
    __shared__ float2 table[TABLE];
    __shared__ float red[GROUPS][LPR * 8];
    const int sub = threadIdx.x % LPR, grp = threadIdx.x / LPR;
    const bool in = 8 * sub < p.D;
    int c0 = 0, c1 = 4;
    if (in) lane_channels<HALF>(p, sub, c0, c1);
    const float inv_d = 1.f / (float)p.D;
    float w[2][8], dw[2][8];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int j = 0; j < 8; ++j) { w[which][j] = 1.f; dw[which][j] = 0.f; }
        if (p.w[which]) load_weight(p, which, c0, c1, w[which]);
    }
    for (long t0 = (long)blockIdx.x * p.tb; t0 < p.tokens; t0 += (long)gridDim.x * p.tb) {
        const int ntok = (int)min((long)p.tb, p.tokens - t0);
        __syncthreads();                                       // the previous tile's rows are done with the table
        fill_table(p, table, t0, ntok);
        __syncthreads();
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const int heads = p.heads[which];
            const bool norm = p.w[which] != nullptr;
            const T* x = reinterpret_cast<const T*>(p.x[which]) + t0 * p.x_ss[which];
            const T* gy = reinterpret_cast<const T*>(p.gy[which]) + t0 * p.g_ss[which];
            T* dx = reinterpret_cast<T*>(p.y[which]) + t0 * heads * (long)p.D;
            const int rows = ntok * heads;
            for (int r0 = grp; r0 < rows; r0 += GROUPS * U) {
                Raw8<T, HALF> rx[U], rg[U];
                int tl[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int r = min(r0 + u * GROUPS, rows - 1);
                    tl[u] = heads == 1 ? r : (int)__umulhi((unsigned)r, p.magic[which]);
                    const int hd = r - tl[u] * heads;
                    if (norm) rx[u].load(x + tl[u] * p.x_ss[which] + hd * p.x_sh[which], c0, c1);
                    rg[u].load(gy + tl[u] * p.g_ss[which] + hd * p.g_sh[which], c0, c1);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int r = r0 + u * GROUPS;
                    const bool live = in && r < rows;
                    float f[8], g[8];
                    rg[u].unpack(g);
                    rotate<HALF>(g, table + tl[u] * p.pairs, 4 * sub, p.pairs);
                    if (norm) {
                        rx[u].unpack(f);
                        float ss = 0.f, dot = 0.f;             // sum x^2 and sum u x:  mean(u xhat) = r * dot / D
#pragma unroll
                        for (int j = 0; j < 8; ++j) { ss += f[j] * f[j]; dot += g[j] * w[which][j] * f[j]; }
                        ss = group_sum<LPR>(in ? ss : 0.f); dot = group_sum<LPR>(in ? dot : 0.f);
                        const float rstd = rsqrtf(ss * inv_d + p.eps), m = rstd * dot * inv_d;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float xh = f[j] * rstd;
                            dw[which][j] += live ? g[j] * xh : 0.f;
                            g[j] = rstd * (g[j] * w[which][j] - xh * m);
                        }
                    }
                    rg[u].pack(g);
                    if (live) rg[u].store(dx + (long)r * p.D, c0, c1);
                }
            }
        }
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        __syncthreads();
        if (in) {
#pragma unroll
            for (int j = 0; j < 4; ++j) { red[grp][c0 + j] = dw[which][j]; red[grp][c1 + j] = dw[which][4 + j]; }
        }
        __syncthreads();
        if ((int)threadIdx.x < p.D) {
            float s = 0.f;
            for (int g = 0; g < GROUPS; ++g) s += red[g][threadIdx.x];
            p.part[((long)blockIdx.x * 2 + which) * p.D + threadIdx.x] = s;
        }
    }
}

// dw[c] (+)= sum over `blocks` partial rows, in a fixed order: 32 columns x 8 slices of rows per workgroup
__global__ void __launch_bounds__(NB) rope_axes_dw_kernel(const float* __restrict__ part, void* dq, void* dk, int q_f32, int k_f32, int accumulate_q, int accumulate_k,
                                                          int blocks, int D) {
    __shared__ float red[8][32];
    const int ct = threadIdx.x & 31, sl = threadIdx.x >> 5, c = blockIdx.x * 32 + ct, which = blockIdx.y;
    float a = 0.f;
    if (c < D) {
#pragma unroll 16
        for (int s = sl; s < blocks; s += 8) a += part[((long)s * 2 + which) * D + c];
    }
    red[sl][ct] = a;
    __syncthreads();
    void* out = which ? dk : dq;
    if (threadIdx.x < 32 && c < D && out) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) s += red[r][ct];
        const bool f32 = which ? k_f32 : q_f32, acc = which ? accumulate_k : accumulate_q;
        if (f32) { float* o = reinterpret_cast<float*>(out) + c; *o = acc ? *o + s : s; }
        else { bf16_t* o = reinterpret_cast<bf16_t*>(out) + c; *o = f32_to_bf16(acc ? bf16_to_f32(*o) + s : s); }
    }
}

// tokens per workgroup: as many as the table holds, while 1 024 workgroups (4 per CU) are left
int tile_tokens(long tokens, int pairs, int D, int heads) {
    int tb = pairs > 0 ? TABLE / pairs : 8;
    if (tb > 8) tb = 8;
    while (tb > 1 && (tokens + tb - 1) / tb < 1024) --tb;
    while (tb > 1 && (long)tb * heads > 65535) --tb;          // row / heads by multiplication
    return tb;
}

bool rows_ok(const void* p, long ss, long sh) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ss % 8 == 0 && sh % 8 == 0; }

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
    if ((wq && wq_dt != DPIPE_BF16 && wq_dt != DPIPE_F32) || (wk && wk_dt != DPIPE_BF16 && wk_dt != DPIPE_F32)) return bad("weights must be bf16 or fp32");
    p.x[0] = q; p.x[1] = k; p.x_ss[0] = q_ss; p.x_sh[0] = q_sh; p.x_ss[1] = k_ss; p.x_sh[1] = k_sh;
    p.pos = pos; p.pos_type = pos_type; p.tokens = tokens; p.period = period; p.axes = axes; p.pairs = pairs; p.D = D;
    p.heads[0] = heads_q; p.heads[1] = heads_k; p.w[0] = wq; p.w[1] = heads_k > 0 ? wk : nullptr;
    p.w_f32[0] = wq_dt == DPIPE_F32; p.w_f32[1] = wk_dt == DPIPE_F32; p.eps = eps;
    for (int w = 0; w < 2; ++w) p.magic[w] = p.heads[w] > 1 ? (unsigned)((0x100000000ull + p.heads[w] - 1) / p.heads[w]) : 0u;
    for (int i = 0; i < pairs; ++i) {
        if (axis[i] < 0 || axis[i] >= axes) return bad("axis index out of range");
        p.freq[i] = freq[i]; p.axis[i] = (unsigned char)axis[i];
    }
    p.tb = tile_tokens(tokens, pairs, D, heads_q > heads_k ? heads_q : heads_k);
    return DPIPE_OK;
}

template <typename T, int LPR> void launch_fwd(const RopeAxesParams& p, bool half, unsigned grid, hipStream_t s) {
    const bool norm = p.w[0] || p.w[1];
    if (half) { if (norm) rope_axes_kernel<T, LPR, true, true><<<grid, NB, 0, s>>>(p); else rope_axes_kernel<T, LPR, true, false><<<grid, NB, 0, s>>>(p); }
    else { if (norm) rope_axes_kernel<T, LPR, false, true><<<grid, NB, 0, s>>>(p); else rope_axes_kernel<T, LPR, false, false><<<grid, NB, 0, s>>>(p); }
}
template <typename T> void launch_fwd(const RopeAxesParams& p, bool half, hipStream_t s) {
    const unsigned grid = (unsigned)cdiv(p.tokens, p.tb);
    if (p.D <= 64) launch_fwd<T, 8>(p, half, grid, s); else if (p.D <= 128) launch_fwd<T, 16>(p, half, grid, s); else launch_fwd<T, 32>(p, half, grid, s);
}
template <typename T> void launch_bwd(const RopeAxesParams& p, bool half, unsigned grid, hipStream_t s) {
#define LAUNCH(LPR) do { if (half) rope_axes_bwd_kernel<T, LPR, true><<<grid, NB, 0, s>>>(p); else rope_axes_bwd_kernel<T, LPR, false><<<grid, NB, 0, s>>>(p); } while (0)
    if (p.D <= 64) LAUNCH(8); else if (p.D <= 128) LAUNCH(16); else LAUNCH(32);
#undef LAUNCH
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
    if (dtype == DPIPE_BF16) launch_fwd<bf16_t>(p, half, reinterpret_cast<hipStream_t>(stream)); else launch_fwd<float>(p, half, reinterpret_cast<hipStream_t>(stream));
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
    if (!gq || (heads_k > 0 && !gk) || !rows_ok(gq, gq_ss, gq_sh) || (heads_k > 0 && !rows_ok(gk, gk_ss, gk_sh)) || !dq || (heads_k > 0 && !dk) || !aligned16(dq) || !aligned16(dk)) {
        set_last_error("dpipe_rope_axes_bwd: gradients must be 16-byte aligned with strides multiple of 8 elements"); return DPIPE_ERR_ARG; }
    const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
    p.y[0] = dq; p.y[1] = dk; p.sign = -1.f;
    if (!p.w[0] && !p.w[1]) {                                  // no norm: the inverse rotation of the gradient
        p.x[0] = gq; p.x[1] = gk; p.x_ss[0] = gq_ss; p.x_sh[0] = gq_sh; p.x_ss[1] = gk_ss; p.x_sh[1] = gk_sh;
        if (dtype == DPIPE_BF16) launch_fwd<bf16_t>(p, half, s); else launch_fwd<float>(p, half, s);
        return check_launch("dpipe_rope_axes_bwd");
    }
    if (!ws) { set_last_error("dpipe_rope_axes_bwd: a normed row needs the workspace"); return DPIPE_ERR_ARG; }
    p.gy[0] = gq; p.gy[1] = gk; p.g_ss[0] = gq_ss; p.g_sh[0] = gq_sh; p.g_ss[1] = gk_ss; p.g_sh[1] = gk_sh; p.part = ws;
    const long tiles = cdiv(tokens, p.tb);
    const unsigned grid = (unsigned)(tiles < MAX_BWD_BLOCKS ? tiles : MAX_BWD_BLOCKS);
    if (dtype == DPIPE_BF16) launch_bwd<bf16_t>(p, half, grid, s); else launch_bwd<float>(p, half, grid, s);
    if (dwq || dwk)
        rope_axes_dw_kernel<<<dim3((unsigned)cdiv(D, 32), 2), NB, 0, s>>>(ws, dwq, dwk, wq_dtype == DPIPE_F32, wk_dtype == DPIPE_F32, accumulate_wq, accumulate_wk, (int)grid, D);
    return check_launch("dpipe_rope_axes_bwd");
}

}  // extern "C"
