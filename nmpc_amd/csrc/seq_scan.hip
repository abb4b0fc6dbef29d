// Selective state-space scan: the linear parameter-varying recurrence with a diagonal state matrix, for every channel d
// (N states, one input u, one output) and step t of a sequence
//   delta = softplus(dt + dt_bias)   (or dt + dt_bias),
//   x_t = exp(delta A) x_{t-1} + delta B_t u_t,      y_t = C_t . x_t + D u_t,      out = y_t silu(z_t).
// Adjoint, with g_t = dout silu(z), lam_t = C_t g_t + exp(delta_{t+1} A) lam_{t+1} and h_t = exp(delta A) x_{t-1}:
//   ddelta = sum_n lam (A h + B u),  du = D g + delta sum_n lam B,  dA = sum_t lam h delta,  dB = sum_d lam delta u,
//   dC = sum_d x g,  dz = dout y silu'(z),  ddt = ddelta softplus'.
//
// Layout.  A lane owns four states of a channel and P = ceil(N / 4) rounded up to 1, 2, 4, 8, 16 lanes a channel (states past N
// are zero throughout); a workgroup of 256 threads owns 256 / P channels of one group (the channels that share B and C) and walks
// the steps in tiles of 32.  A tile's samples are staged once per element through LDS (softplus, its product with u), so that the
// P lanes of a channel do not repeat them; B and C are read from LDS as one 16-byte access per lane.
// What bounds it: VALU issue.  A state and step costs 2 (exp2) + 4 slots forward; the bytes are 8 a channel and step in bf16.
#include <algorithm>

#include "seq_common.h"

namespace nmpc {

constexpr int SCAN_T = 32;             // steps of a tile
constexpr int SCAN_THREADS = 256;

struct ScanDev {
    nmpc_scan_args a;
    int nblk, per;                     // channel blocks of a group, channels of a group
    int ntile, nch, tpc;               // tiles; chunks (parts of the time axis that run side by side) and tiles of a chunk
    float *xin, *dsum;                 // [nb][nch][D][4P] state before a chunk; [nb][nch][D] sum of delta over it
    float *pA, *pDb, *pBC;             // partial sums (backward)
};

__device__ __forceinline__ float softplus(float x) {
    if (x > 20.f) return x;            // e^-20 is below half a step of x
    return log1pf(__builtin_amdgcn_exp2f(x * LOG2E));
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true);
    return v + __builtin_bit_cast(float, o);
}
// sum over the P lanes of a channel; every lane gets the same bits
template <int P>
__device__ __forceinline__ float sum_lanes(float v) {
    if constexpr (P >= 2) v = dpp_add<0xB1>(v);       // quad_perm [1,0,3,2]
    if constexpr (P >= 4) v = dpp_add<0x4E>(v);       // quad_perm [2,3,0,1]
    if constexpr (P >= 8) v = dpp_add<0x141>(v);      // mirror within 8
    if constexpr (P >= 16) v = dpp_add<0x140>(v);     // mirror within 16
    return v;
}

// Where a workgroup works: channel block of a group, chunk, sequence.
template <int P>
struct ScanPlace {
    static constexpr int CH = SCAN_THREADS / P;
    int b, chunk, g, c0, nvalid, len;                 // first channel, channels that exist
    __device__ __forceinline__ ScanPlace(const ScanDev& s) {
        const int nb_x = s.a.G * s.nblk;
        const int blk = blockIdx.x % nb_x, rest = blockIdx.x / nb_x;
        chunk = rest % s.nch; b = rest / s.nch;
        g = blk / s.nblk;
        const int first = (blk % s.nblk) * CH;
        c0 = g * s.per + first;
        nvalid = min(CH, s.per - first);
        len = seq_length(s.a.lengths, b, s.a.L);
    }
};

// rows t0 .. t0+31 of B or C (of this group) as fp32, zero past the sequence and past N
template <typename T, int P>
__device__ __forceinline__ void stage_bc(float (*dst)[4 * P], const void* src, long long bs, long long ts, int b, int g, int N, int t0, int len) {
    const T* p = (const T*)src + b * bs + (long long)g * N;
    for (int e = threadIdx.x; e < SCAN_T * 4 * P; e += SCAN_THREADS) {
        const int t = e / (4 * P), n = e % (4 * P);
        dst[t][n] = (t0 + t < len && n < N) ? (float)p[(long long)(t0 + t) * ts + n] : 0.f;
    }
}

template <int P>
__device__ __forceinline__ void load_A(const ScanDev& s, int c, bool ok, int q, float (&a)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = 4 * q + i;
        a[i] = ok && n < s.a.N ? s.a.A[(long long)c * s.a.N + n] * LOG2E : 0.f;
    }
}

// four states of a channel in an array [..][N]
__device__ __forceinline__ void load_states(const float* p, int N, int q, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = 4 * q + i < N ? p[4 * q + i] : 0.f;
}
__device__ __forceinline__ void store_states(float* p, int N, int q, const float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (4 * q + i < N) p[4 * q + i] = x[i];
}

// SUMMARY: only what the steps of a chunk do to a state: x_end = exp2(a dsum) x_begin + xin, started from zero.
// Otherwise the scan itself from the state before the chunk.
template <typename T, int P, bool SUMMARY>
__global__ __launch_bounds__(SCAN_THREADS) void scan_fwd_kernel(ScanDev s) {
    constexpr int CH = SCAN_THREADS / P;
    __shared__ float2 sDX[SCAN_T][CH];                // delta, delta u
    __shared__ float sB[SCAN_T][4 * P], sC[SUMMARY ? 1 : SCAN_T][4 * P], sY[SUMMARY ? 1 : SCAN_T][CH];
    const nmpc_scan_args& a = s.a;
    const ScanPlace<P> at(s);
    const int tid = threadIdx.x, c = tid / P, q = tid % P, ch = at.c0 + c;
    const bool ok = c < at.nvalid;
    float A[4], x[4] = {0.f, 0.f, 0.f, 0.f}, total = 0.f;
    load_A<P>(s, ch, ok, q, A);
    const long long part = ((long long)(at.b * s.nch + at.chunk) * a.D + ch) * (4 * P) + 4 * q;
    if (!SUMMARY && ok) {
        if (s.nch > 1) load_states(s.xin + part - 4 * q, 4 * P, q, x);
        else if (a.start) load_states(a.start + ((long long)at.b * a.D + ch) * a.N, a.N, q, x);
    }
    const T* u = (const T*)a.u + at.b * a.u_bs + at.c0;
    const T* dt = (const T*)a.dt + at.b * a.dt_bs + at.c0;
    const T* z = a.z ? (const T*)a.z + at.b * a.z_bs + at.c0 : nullptr;
    const int tile0 = at.chunk * s.tpc, tile1 = min(tile0 + s.tpc, s.ntile);
    for (int tile = tile0; tile < tile1; ++tile) {
        const int t0 = tile * SCAN_T;
        __syncthreads();
        for (int e = tid; e < SCAN_T * CH; e += SCAN_THREADS) {
            const int t = e / CH, cc = e % CH;
            float d = 0.f, du = 0.f;
            if (t0 + t < at.len && cc < at.nvalid) {
                d = (float)dt[(long long)(t0 + t) * a.dt_ts + cc] + (a.dt_bias ? a.dt_bias[at.c0 + cc] : 0.f);
                if (a.softplus) d = softplus(d);
                du = d * (float)u[(long long)(t0 + t) * a.u_ts + cc];
            }
            sDX[t][cc] = make_float2(d, du);
        }
        stage_bc<T, P>(sB, a.B, a.B_bs, a.B_ts, at.b, at.g, a.N, t0, at.len);
        if constexpr (!SUMMARY) {
            stage_bc<T, P>(sC, a.C, a.C_bs, a.C_ts, at.b, at.g, a.N, t0, at.len);
            if (a.saved && ok) store_states((float*)a.saved + (((long long)at.b * s.ntile + tile) * a.D + ch) * (4 * P), 4 * P, q, x);
        }
        __syncthreads();
#pragma unroll 4
        for (int t = 0; t < SCAN_T; ++t) {
            const float2 dx = sDX[t][c];
            const float4 b4 = *reinterpret_cast<const float4*>(&sB[t][4 * q]);
            const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_exp2f(dx.x * A[i]) * x[i] + dx.y * b[i];
            if constexpr (SUMMARY) {
                total += dx.x;
            } else {
                const float4 c4 = *reinterpret_cast<const float4*>(&sC[t][4 * q]);
                const float y = sum_lanes<P>(c4.x * x[0] + c4.y * x[1] + c4.z * x[2] + c4.w * x[3]);
                if (q == 0) sY[t][c] = y;
            }
        }
        if constexpr (!SUMMARY) {
            __syncthreads();
            T* y = (T*)a.y + ((long long)at.b * a.L + t0) * a.D + at.c0;
            for (int e = tid; e < SCAN_T * CH; e += SCAN_THREADS) {
                const int t = e / CH, cc = e % CH;
                if (t0 + t >= a.L || cc >= at.nvalid) continue;
                float v = 0.f;
                if (t0 + t < at.len) {
                    v = sY[t][cc];
                    if (a.D_skip) v += a.D_skip[at.c0 + cc] * (float)u[(long long)(t0 + t) * a.u_ts + cc];
                    if (z) {
                        const float zz = (float)z[(long long)(t0 + t) * a.z_ts + cc];
                        v *= zz * sigmoid(zz);
                    }
                }
                y[(long long)t * a.D + cc] = (T)v;
            }
        }
    }
    if (!ok) return;
    if constexpr (SUMMARY) {
        store_states(s.xin + part - 4 * q, 4 * P, q, x);
        if (q == 0) s.dsum[(long long)(at.b * s.nch + at.chunk) * a.D + ch] = total;
    } else if (a.last && at.chunk == s.nch - 1) {
        store_states(a.last + ((long long)at.b * a.D + ch) * a.N, a.N, q, x);
    }
}

// From the chunks' summaries to the state before every chunk (REVERSE: the adjoint behind every chunk), in place.
template <bool REVERSE>
__global__ __launch_bounds__(256) void scan_chunks_kernel(ScanDev s, int NP) {
    const nmpc_scan_args& a = s.a;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x;
    const int n = (int)(id % NP);
    const long long bc = id / NP;
    const int ch = (int)(bc % a.D), b = (int)(bc / a.D);
    if (b >= a.nb) return;
    const float A = n < a.N ? a.A[(long long)ch * a.N + n] * LOG2E : 0.f;
    const float* begin = REVERSE ? a.dlast : a.start;
    float x = begin && n < a.N ? begin[((long long)b * a.D + ch) * a.N + n] : 0.f;
    for (int k = 0; k < s.nch; ++k) {
        const long long at = (long long)b * s.nch + (REVERSE ? s.nch - 1 - k : k);
        float* p = s.xin + (at * a.D + ch) * NP + n;
        const float own = *p;
        *p = x;
        x = __builtin_amdgcn_exp2f(A * s.dsum[at * a.D + ch]) * x + own;
    }
}

// The adjoint's summary of a chunk: lam before its first step, times that step's decay, started from zero behind its last.
template <typename T, int P>
__global__ __launch_bounds__(SCAN_THREADS) void scan_bwd_summary_kernel(ScanDev s) {
    constexpr int CH = SCAN_THREADS / P;
    __shared__ float2 sDG[SCAN_T][CH];                // delta, g
    __shared__ float sC[SCAN_T][4 * P];
    const nmpc_scan_args& a = s.a;
    const ScanPlace<P> at(s);
    const int tid = threadIdx.x, c = tid / P, q = tid % P, ch = at.c0 + c;
    const bool ok = c < at.nvalid;
    float A[4], lam[4] = {0.f, 0.f, 0.f, 0.f}, total = 0.f;
    load_A<P>(s, ch, ok, q, A);
    const T* dt = (const T*)a.dt + at.b * a.dt_bs + at.c0;
    const T* z = a.z ? (const T*)a.z + at.b * a.z_bs + at.c0 : nullptr;
    const T* dy = (const T*)a.dy + at.b * a.dy_bs + at.c0;
    const int tile0 = at.chunk * s.tpc, tile1 = min(tile0 + s.tpc, s.ntile);
    for (int tile = tile1 - 1; tile >= tile0; --tile) {
        const int t0 = tile * SCAN_T;
        __syncthreads();
        for (int e = tid; e < SCAN_T * CH; e += SCAN_THREADS) {
            const int t = e / CH, cc = e % CH;
            float d = 0.f, g = 0.f;
            if (t0 + t < at.len && cc < at.nvalid) {
                d = (float)dt[(long long)(t0 + t) * a.dt_ts + cc] + (a.dt_bias ? a.dt_bias[at.c0 + cc] : 0.f);
                if (a.softplus) d = softplus(d);
                g = (float)dy[(long long)(t0 + t) * a.dy_ts + cc];
                if (z) {
                    const float zz = (float)z[(long long)(t0 + t) * a.z_ts + cc];
                    g *= zz * sigmoid(zz);
                }
            }
            sDG[t][cc] = make_float2(d, g);
        }
        stage_bc<T, P>(sC, a.C, a.C_bs, a.C_ts, at.b, at.g, a.N, t0, at.len);
        __syncthreads();
#pragma unroll 4
        for (int t = SCAN_T - 1; t >= 0; --t) {
            const float2 dg = sDG[t][c];
            const float4 c4 = *reinterpret_cast<const float4*>(&sC[t][4 * q]);
            const float C[4] = {c4.x, c4.y, c4.z, c4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) lam[i] = (lam[i] + C[i] * dg.y) * __builtin_amdgcn_exp2f(dg.x * A[i]);
            total += dg.x;
        }
    }
    if (!ok) return;
    store_states(s.xin + ((long long)(at.b * s.nch + at.chunk) * a.D + ch) * (4 * P), 4 * P, q, lam);
    if (q == 0) s.dsum[(long long)(at.b * s.nch + at.chunk) * a.D + ch] = total;
}

// Tiles from the last to the first: the states of a tile are recomputed from the one saved before it and stay in registers,
// then the adjoint runs back through them.
template <typename T, int P>
__global__ __launch_bounds__(SCAN_THREADS, P == 1 || P == 16 ? 1 : 2) void scan_bwd_kernel(ScanDev s) {
    constexpr int CH = SCAN_THREADS / P, NP = 4 * P;
    __shared__ float2 sDU[SCAN_T][CH];                // delta, u;  afterwards sum_n lam B, sum_n lam h A log2(e)
    __shared__ float sG[SCAN_T][CH], sY[SCAN_T][CH];
    __shared__ float sB[SCAN_T][NP], sC[SCAN_T][NP];
    __shared__ float sP[4][SCAN_T][2 * NP];           // each wave's sums of dB, dC over its channels
    const nmpc_scan_args& a = s.a;
    const ScanPlace<P> at(s);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = tid / P, q = tid % P, ch = at.c0 + c;
    const bool ok = c < at.nvalid;
    float A[4], lam[4] = {0.f, 0.f, 0.f, 0.f}, dA[4] = {0.f, 0.f, 0.f, 0.f}, dD = 0.f, db = 0.f;
    load_A<P>(s, ch, ok, q, A);
    const long long row = (long long)at.b * s.nch + at.chunk;
    if (ok) {
        if (s.nch > 1) load_states(s.xin + (row * a.D + ch) * NP, NP, q, lam);
        else if (a.dlast) load_states(a.dlast + ((long long)at.b * a.D + ch) * a.N, a.N, q, lam);
    }
    const T* u = (const T*)a.u + at.b * a.u_bs + at.c0;
    const T* dt = (const T*)a.dt + at.b * a.dt_bs + at.c0;
    const T* z = a.z ? (const T*)a.z + at.b * a.z_bs + at.c0 : nullptr;
    const T* dy = (const T*)a.dy + at.b * a.dy_bs + at.c0;
    const long long out0 = (long long)at.b * a.L * a.D + at.c0;
    const int tile0 = at.chunk * s.tpc, tile1 = min(tile0 + s.tpc, s.ntile);
    for (int tile = tile1 - 1; tile >= tile0; --tile) {
        const int t0 = tile * SCAN_T;
        __syncthreads();
        for (int e = tid; e < SCAN_T * CH; e += SCAN_THREADS) {
            const int t = e / CH, cc = e % CH;
            float d = 0.f, uu = 0.f, g = 0.f;
            if (t0 + t < at.len && cc < at.nvalid) {
                d = (float)dt[(long long)(t0 + t) * a.dt_ts + cc] + (a.dt_bias ? a.dt_bias[at.c0 + cc] : 0.f);
                if (a.softplus) d = softplus(d);
                uu = (float)u[(long long)(t0 + t) * a.u_ts + cc];
                g = (float)dy[(long long)(t0 + t) * a.dy_ts + cc];
                if (z) {
                    const float zz = (float)z[(long long)(t0 + t) * a.z_ts + cc];
                    g *= zz * sigmoid(zz);
                }
            }
            sDU[t][cc] = make_float2(d, uu);
            sG[t][cc] = g;
        }
        stage_bc<T, P>(sB, a.B, a.B_bs, a.B_ts, at.b, at.g, a.N, t0, at.len);
        stage_bc<T, P>(sC, a.C, a.C_bs, a.C_ts, at.b, at.g, a.N, t0, at.len);
        float x0[4] = {0.f, 0.f, 0.f, 0.f}, xs[SCAN_T][4];
        if (ok) load_states((const float*)a.saved + (((long long)at.b * s.ntile + tile) * a.D + ch) * NP, NP, q, x0);
        __syncthreads();
#pragma unroll
        for (int t = 0; t < SCAN_T; ++t) {
            const float2 du = sDU[t][c];
            const float4 b4 = *reinterpret_cast<const float4*>(&sB[t][4 * q]);
            const float b[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                xs[t][i] = __builtin_amdgcn_exp2f(du.x * A[i]) * (t ? xs[t - 1][i] : x0[i]) + (du.x * du.y) * b[i];
            if (z) {
                const float4 c4 = *reinterpret_cast<const float4*>(&sC[t][4 * q]);
                const float y = sum_lanes<P>(c4.x * xs[t][0] + c4.y * xs[t][1] + c4.z * xs[t][2] + c4.w * xs[t][3]);
                if (q == 0) sY[t][c] = y;
            }
        }
#pragma unroll
        for (int t = SCAN_T - 1; t >= 0; --t) {
            const float2 du = sDU[t][c];
            const float g = sG[t][c], w = du.x * du.y;
            const float4 b4 = *reinterpret_cast<const float4*>(&sB[t][4 * q]), c4 = *reinterpret_cast<const float4*>(&sC[t][4 * q]);
            const float b[4] = {b4.x, b4.y, b4.z, b4.w}, C[4] = {c4.x, c4.y, c4.z, c4.w};
            float s1 = 0.f, s2 = 0.f, p[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(du.x * A[i]);
                lam[i] += C[i] * g;
                p[i] = lam[i] * w;
                p[4 + i] = xs[t][i] * g;
                s1 += lam[i] * b[i];
                lam[i] *= e;
                const float m = lam[i] * (t ? xs[t > 0 ? t - 1 : 0][i] : x0[i]);
                s2 += m * A[i];
                dA[i] += m * du.x;
            }
            s1 = sum_lanes<P>(s1);
            s2 = sum_lanes<P>(s2);
            // all lanes of the channel have read this entry (they are in one wave)
            if (q == 0) sDU[t][c] = make_float2(s1, s2);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
                for (int m = P; m < 64; m *= 2) p[i] += __shfl_xor(p[i], m);
            }
            if (lane < P) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sP[wave][t][4 * q + i] = p[i];
                    sP[wave][t][NP + 4 * q + i] = p[4 + i];
                }
            }
        }
        __syncthreads();
        for (int e = tid; e < SCAN_T * 2 * NP; e += SCAN_THREADS) {
            const int t = e / (2 * NP), n = e % (2 * NP);
            if (t0 + t >= a.L) continue;
            const float v = (sP[0][t][n] + sP[1][t][n]) + (sP[2][t][n] + sP[3][t][n]);
            const long long blk = (at.c0 - at.g * s.per) / CH;
            s.pBC[(((blk * a.nb + at.b) * a.L + t0 + t) * a.G + at.g) * (2 * NP) + n] = v;
        }
        for (int e = tid; e < SCAN_T * CH; e += SCAN_THREADS) {
            const int t = e / CH, cc = e % CH;
            if (t0 + t >= a.L || cc >= at.nvalid) continue;
            const long long o = out0 + (long long)(t0 + t) * a.D + cc;
            float vu = 0.f, vd = 0.f, vz = 0.f;
            if (t0 + t < at.len) {
                const float2 sums = sDU[t][cc];
                const float raw = (float)dt[(long long)(t0 + t) * a.dt_ts + cc] + (a.dt_bias ? a.dt_bias[at.c0 + cc] : 0.f);
                const float d = a.softplus ? softplus(raw) : raw, uu = (float)u[(long long)(t0 + t) * a.u_ts + cc], g = sG[t][cc];
                const float skip = a.D_skip ? a.D_skip[at.c0 + cc] : 0.f;
                vu = skip * g + d * sums.x;
                vd = sums.y * (1.f / LOG2E) + uu * sums.x;
                if (a.softplus) vd *= sigmoid(raw);
                if (z) {
                    const float zz = (float)z[(long long)(t0 + t) * a.z_ts + cc], p = sigmoid(zz);
                    vz = (float)dy[(long long)(t0 + t) * a.dy_ts + cc] * (sY[t][cc] + skip * uu) * (p * (1.f + zz * (1.f - p)));
                }
                dD += g * uu;
                db += vd;
            }
            ((T*)a.du)[o] = (T)vu;
            ((T*)a.ddt)[o] = (T)vd;
            if (z) ((T*)a.dz)[o] = (T)vz;
        }
    }
    if (ok) {
        store_states(s.pA + (row * a.D + ch) * NP, NP, q, dA);
        if (a.dstart && at.chunk == 0) store_states(a.dstart + ((long long)at.b * a.D + ch) * a.N, a.N, q, lam);
    }
    // dD and the bias: a thread's elements are all of channel tid % CH
    __syncthreads();
    float* red = &sG[0][0];
    red[tid] = dD;
    red[SCAN_THREADS + tid] = db;
    __syncthreads();
    if (tid < at.nvalid) {
        float v0 = 0.f, v1 = 0.f;
        for (int r = tid; r < SCAN_THREADS; r += CH) { v0 += red[r]; v1 += red[SCAN_THREADS + r]; }
        s.pDb[(row * 2) * a.D + at.c0 + tid] = v0;
        s.pDb[(row * 2 + 1) * a.D + at.c0 + tid] = v1;
    }
}

// Sums of the partial sums over sequences and chunks (dA, dD, the bias) and over channel blocks (dB, dC), in a fixed order.
__global__ __launch_bounds__(256) void scan_reduce_params_kernel(ScanDev s, int NP) {
    const nmpc_scan_args& a = s.a;
    const long long rows = (long long)a.nb * s.nch, id = (long long)blockIdx.x * 256 + threadIdx.x, nA = (long long)a.D * NP;
    if (id < nA) {
        float v = 0.f;
        for (long long r = 0; r < rows; ++r) v += s.pA[r * nA + id];
        const int n = (int)(id % NP);
        if (n < a.N) a.dA[(id / NP) * a.N + n] = v;
    } else if (id < nA + 2 * a.D) {
        const int k = (int)((id - nA) / a.D), ch = (int)((id - nA) % a.D);
        float* out = k ? a.ddt_bias : a.dD;
        if (!out) return;
        float v = 0.f;
        for (long long r = 0; r < rows; ++r) v += s.pDb[(r * 2 + k) * a.D + ch];
        out[ch] = v;
    }
}
template <typename T>
__global__ __launch_bounds__(256) void scan_reduce_bc_kernel(ScanDev s, int NP) {
    const nmpc_scan_args& a = s.a;
    const long long rows = (long long)a.nb * a.L * a.G;
    for (long long id = (long long)blockIdx.x * 256 + threadIdx.x; id < rows * 2 * NP; id += 256ll * gridDim.x) {
        const int n = (int)(id % (2 * NP));
        const long long r = id / (2 * NP);
        float v = 0.f;
        for (int k = 0; k < s.nblk; ++k) v += s.pBC[(k * rows + r) * (2 * NP) + n];
        if (n < a.N) ((T*)a.dB)[r * a.N + n] = (T)v;
        else if (n >= NP && n - NP < a.N) ((T*)a.dC)[r * a.N + n - NP] = (T)v;
    }
}

// One step of every sequence; the state a.last is read and replaced.
template <typename T, int P>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanDev s) {
    const nmpc_scan_args& a = s.a;
    const long long id = (long long)blockIdx.x * 256 + threadIdx.x, bc = id / P;
    const int q = (int)(id % P), b = (int)(bc / a.D), ch = (int)(bc % a.D);
    if (b >= a.nb) return;                            // the P lanes of a channel leave together
    const int g = ch / s.per;
    float A[4], x[4];
    load_A<P>(s, ch, true, q, A);
    float* state = a.last + bc * a.N;
    load_states(state, a.N, q, x);
    const float uu = (float)((const T*)a.u)[b * a.u_bs + ch];
    float d = (float)((const T*)a.dt)[b * a.dt_bs + ch] + (a.dt_bias ? a.dt_bias[ch] : 0.f);
    if (a.softplus) d = softplus(d);
    const T* Bp = (const T*)a.B + b * a.B_bs + (long long)g * a.N;
    const T* Cp = (const T*)a.C + b * a.C_bs + (long long)g * a.N;
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = 4 * q + i;
        if (n < a.N) {
            x[i] = __builtin_amdgcn_exp2f(d * A[i]) * x[i] + (d * uu) * (float)Bp[n];
            y += (float)Cp[n] * x[i];
        }
    }
    store_states(state, a.N, q, x);
    y = sum_lanes<P>(y);
    if (q == 0) {
        if (a.D_skip) y += a.D_skip[ch] * uu;
        if (a.z) {
            const float zz = (float)((const T*)a.z)[b * a.z_bs + ch];
            y *= zz * sigmoid(zz);
        }
        ((T*)a.y)[bc] = (T)y;
    }
}

static int scan_lanes(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

static void scan_plan(ScanDev& s) {
    const nmpc_scan_args& a = s.a;
    const int P = scan_lanes(a.N), CH = SCAN_THREADS / P;
    s.per = a.D / a.G;
    s.nblk = (s.per + CH - 1) / CH;
    s.ntile = a.L > 0 ? (a.L + SCAN_T - 1) / SCAN_T : 0;
    s.nch = 1;
    s.tpc = s.ntile;
}

static unsigned long long round256(unsigned long long v) { return (v + 255) / 256 * 256; }

// lays the workspace out; returns its bytes
static unsigned long long scan_workspace(ScanDev& s, bool backward, char* base) {
    const nmpc_scan_args& a = s.a;
    const unsigned long long NP = 4 * scan_lanes(a.N), rows = (unsigned long long)a.nb * s.nch;
    unsigned long long off = 0;
    auto take = [&](float*& p, unsigned long long floats) { p = (float*)(base + off); off += round256(floats * 4); };
    if (s.nch > 1) { take(s.xin, rows * a.D * NP); take(s.dsum, rows * a.D); }
    if (backward) {
        take(s.pA, rows * a.D * NP);
        take(s.pDb, rows * 2 * a.D);
        take(s.pBC, (unsigned long long)s.nblk * a.nb * a.L * a.G * 2 * NP);
    }
    return off;
}

static int scan_check(const char* what, const nmpc_scan_args* a) {
    NMPC_REQUIRE(a, "%s: null argument", what);
    NMPC_REQUIRE(a->struct_size == (int)sizeof(nmpc_scan_args), "%s: struct of %d bytes, the library's has %d", what, a->struct_size,
                 (int)sizeof(nmpc_scan_args));
    NMPC_REQUIRE(a->dtype >= NMPC_F32 && a->dtype <= NMPC_F16, "%s: unknown element type %d", what, a->dtype);
    NMPC_REQUIRE(a->nb >= 0 && a->L >= 0 && a->D >= 1, "%s: bad sizes (%d sequences, %d steps, %d channels)", what, a->nb, a->L, a->D);
    NMPC_REQUIRE(a->N >= 1 && a->N <= 64, "%s: %d states a channel (1..64)", what, a->N);
    NMPC_REQUIRE(a->G >= 1 && a->D % a->G == 0, "%s: %d groups do not divide %d channels", what, a->G, a->D);
    // a launch has fewer than 2^32 threads
    NMPC_REQUIRE((long long)a->nb * a->D * 64 < (1ll << 31) && (long long)a->nb * (a->D / 16 + a->G) * (a->L / SCAN_T + 1) < (1ll << 23),
                 "%s: too many elements for one launch", what);
    return 0;
}

#define NMPC_P_SWITCH(N, ...)                                    \
    switch (scan_lanes(N)) {                                     \
        case 1: { constexpr int P_ = 1; __VA_ARGS__ } break;     \
        case 2: { constexpr int P_ = 2; __VA_ARGS__ } break;     \
        case 4: { constexpr int P_ = 4; __VA_ARGS__ } break;     \
        case 8: { constexpr int P_ = 8; __VA_ARGS__ } break;     \
        default: { constexpr int P_ = 16; __VA_ARGS__ } break;   \
    }

}  // namespace nmpc

using namespace nmpc;

extern "C" unsigned long long nmpc_lpv_scan_saved_bytes(int nb, int L, int D, int N) {
    if (nb <= 0 || L <= 0 || D <= 0 || N <= 0 || N > 64) return 0;
    return (unsigned long long)nb * ((L + SCAN_T - 1) / SCAN_T) * D * 4 * scan_lanes(N) * sizeof(float);
}

extern "C" unsigned long long nmpc_lpv_scan_workspace_bytes(int nb, int L, int D, int N, int G, int backward) {
    if (nb <= 0 || L < 0 || D <= 0 || N <= 0 || N > 64 || G <= 0 || D % G) return 0;
    ScanDev s = {};
    s.a.nb = nb; s.a.L = L; s.a.D = D; s.a.N = N; s.a.G = G;
    scan_plan(s);
    return scan_workspace(s, backward != 0, nullptr);
}

extern "C" int nmpc_lpv_scan(const nmpc_scan_args* args, void* stream) {
    if (scan_check("nmpc_lpv_scan", args)) return 1;
    ScanDev s = {};
    s.a = *args;
    const nmpc_scan_args& a = s.a;
    if (a.nb == 0) return 0;
    NMPC_REQUIRE(a.A && (a.L == 0 || (a.u && a.dt && a.B && a.C && a.y)), "nmpc_lpv_scan: null argument");
    scan_plan(s);
    const unsigned long long need = scan_workspace(s, false, (char*)a.workspace);
    NMPC_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need), "nmpc_lpv_scan: workspace of %llu bytes, %llu needed", a.workspace_bytes, need);
    const unsigned grid = (unsigned)(a.nb * (long long)s.nch * a.G * s.nblk);
    const hipStream_t st = (hipStream_t)stream;
    NMPC_DTYPE_SWITCH(a.dtype, {
        NMPC_P_SWITCH(a.N, {
            if (s.nch > 1) {
                scan_fwd_kernel<T_, P_, true><<<grid, SCAN_THREADS, 0, st>>>(s);
                scan_chunks_kernel<false><<<(unsigned)(((long long)a.nb * a.D * 4 * P_ + 255) / 256), 256, 0, st>>>(s, 4 * P_);
            }
            scan_fwd_kernel<T_, P_, false><<<grid, SCAN_THREADS, 0, st>>>(s);
        })
    })
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int nmpc_lpv_scan_bwd(const nmpc_scan_args* args, void* stream) {
    if (scan_check("nmpc_lpv_scan_bwd", args)) return 1;
    ScanDev s = {};
    s.a = *args;
    const nmpc_scan_args& a = s.a;
    NMPC_REQUIRE(a.A && a.dA, "nmpc_lpv_scan_bwd: null argument");
    NMPC_REQUIRE(a.nb == 0 || a.L == 0 || (a.u && a.dt && a.B && a.C && a.saved && a.dy && a.du && a.ddt && a.dB && a.dC && (!a.z || a.dz)),
                 "nmpc_lpv_scan_bwd: null argument");
    NMPC_REQUIRE(!a.D_skip || a.dD, "nmpc_lpv_scan_bwd: D needs dD");
    NMPC_REQUIRE(!a.dt_bias || a.ddt_bias, "nmpc_lpv_scan_bwd: dt_bias needs ddt_bias");
    scan_plan(s);
    const unsigned long long need = a.nb > 0 ? scan_workspace(s, true, (char*)a.workspace) : 0;
    NMPC_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need), "nmpc_lpv_scan_bwd: workspace of %llu bytes, %llu needed", a.workspace_bytes, need);
    const unsigned grid = (unsigned)(a.nb * (long long)s.nch * a.G * s.nblk);
    const hipStream_t st = (hipStream_t)stream;
    NMPC_DTYPE_SWITCH(a.dtype, {
        NMPC_P_SWITCH(a.N, {
            constexpr int NP = 4 * P_;
            if (a.nb > 0) {
                if (s.nch > 1) {
                    scan_bwd_summary_kernel<T_, P_><<<grid, SCAN_THREADS, 0, st>>>(s);
                    scan_chunks_kernel<true><<<(unsigned)(((long long)a.nb * a.D * NP + 255) / 256), 256, 0, st>>>(s, NP);
                }
                scan_bwd_kernel<T_, P_><<<grid, SCAN_THREADS, 0, st>>>(s);
            }
            scan_reduce_params_kernel<<<(unsigned)(((long long)a.D * (NP + 2) + 255) / 256), 256, 0, st>>>(s, NP);
            const long long nbc = (long long)a.nb * a.L * a.G * 2 * NP;
            if (nbc > 0) scan_reduce_bc_kernel<T_><<<(unsigned)std::min((nbc + 255) / 256, 1ll << 20), 256, 0, st>>>(s, NP);
        })
    })
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int nmpc_lpv_scan_step(const nmpc_scan_args* args, void* stream) {
    if (scan_check("nmpc_lpv_scan_step", args)) return 1;
    ScanDev s = {};
    s.a = *args;
    const nmpc_scan_args& a = s.a;
    if (a.nb == 0) return 0;
    NMPC_REQUIRE(a.A && a.u && a.dt && a.B && a.C && a.y && a.last, "nmpc_lpv_scan_step: null argument");
    scan_plan(s);
    NMPC_DTYPE_SWITCH(a.dtype, {
        NMPC_P_SWITCH(a.N, {
            scan_step_kernel<T_, P_><<<(unsigned)(((long long)a.nb * a.D * P_ + 255) / 256), 256, 0, (hipStream_t)stream>>>(s);
        })
    })
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}
