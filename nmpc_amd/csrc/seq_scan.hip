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
// P lanes of a channel do not repeat them; B and C are read from LDS as one 16-byte access per lane; the next tile's loads are in
// flight meanwhile.  Sequences that do not fill the chip are cut in time (scan_plan): chunks whose effect on a state, x_end =
// exp(A sum delta) x_begin + own, is found in a pass before, or slots of a workgroup that keep their decays in registers.
// What bounds it: VALU issue.  A state and step costs 6.5 slots forward (its exponential alone 2.5) and about 22 backward, of which
// 6.5 are the states of a tile computed again from the one saved before it: saving every 16th state costs 1/4 byte a state and step
// instead of 4.  Sums over the lanes of a channel and over the channels of a group trade
// halves, so that four steps (eight values) share the stages of one.
// Measured, bf16, 16 states: 4 x 2048 steps x 2048 channels forward 124 us, training 483 us (280 of them the main backward pass);
// 1 x 8192 x 2048 forward 152 us; step of 64 x 4096 channels 9.5 us, 3.8 TB/s.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "seq_common.h"

namespace nmpc {

constexpr int SCAN_T = 32;             // steps of a tile
constexpr int SCAN_SAVE = 16;          // the forward pass saves the state before every 16th step: a tile of the backward pass
constexpr int SCAN_THREADS = 256;

struct ScanDev {
    nmpc_scan_args a;
    int nblk, per;                     // channel blocks of a group, channels of a group
    int ntile, nch, tpc;               // tiles; chunks (parts of the time axis that run side by side) and tiles of a chunk
    int slots;                         // forward: the time axis in slots of a workgroup
    float *xin, *dsum;                 // [nb][nch][D][4P] state before a chunk; [nb][nch][D] sum of delta over it
    float *pA, *pDb, *pBC;             // partial sums (backward)
};

// softplus(x) = max(x, 0) + log(1 + e) with e = e^-|x| <= 1, and log(1 + e) = 2 atanh(s), s = e / (2 + e) <= 1/3: a polynomial in s^2
// through the Chebyshev points of [0, 1/9] (off by 8e-9 of the value), so that small values keep their relative accuracy
__device__ __forceinline__ float softplus(float x) {
    const float e = __builtin_amdgcn_exp2f(-LOG2E * fabsf(x)), s = e * __builtin_amdgcn_rcpf(2.f + e), q = s * s;
    const float r = 1.f + q * (0.33333161f + q * (0.20012298f + q * (0.13982579f + q * 0.1407889f)));
    return fmaxf(x, 0.f) + 2.f * s * r;
}

// What many steps do to a state: x 2^e, as three products with 2^(e/3).  A growing mode may grow past any fp32 number on a state so small
// that the result is an ordinary one, or on a state of zero: each factor stays at or below 2^127, and all three carry the smallest number
// past the largest, so that nothing but the result's own overflow is lost.  One factor, which cannot do that, would save 1 .. 2 % of the
// slots kernel (4 x 2048 x 2048, 16 states: 126 instead of 128 us).
__device__ __forceinline__ float growth_root(float e) { return __builtin_amdgcn_exp2f(fminf(e * (1.f / 3.f), 127.f)); }

template <int CTRL, int BANKS = 0xf>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, BANKS, true));
}
constexpr int DPP_XOR1 = 0xB1, DPP_XOR2 = 0x4E, DPP_SHL4 = 0x104, DPP_ROR8 = 0x128, DPP_HALF_MIRROR = 0x141, DPP_MIRROR = 0x140;

// sum over the P lanes of a channel; every lane gets the same bits
template <int P>
__device__ __forceinline__ float sum_lanes(float v) {
    if constexpr (P >= 2) v += dpp<DPP_XOR1>(v);
    if constexpr (P >= 4) v += dpp<DPP_XOR2>(v);
    if constexpr (P >= 8) v += dpp<DPP_HALF_MIRROR>(v);
    if constexpr (P >= 16) v += dpp<DPP_MIRROR>(v);
    return v;
}

// The same for the values of S = min(P, 4) steps at once: lane q < S gets the sum of step q (others: nothing of use).  A lane of a pair
// keeps one of two values and hands the other over, so that each stage halves the values instead of repeating the sum.
template <int P>
struct Steps {
    static constexpr int S = P < 4 ? P : 4;
};
template <int P>
__device__ __forceinline__ float sum_steps(const float (&y)[Steps<P>::S], int lane) {
    if constexpr (P == 1) return y[0];
    else {
        const bool odd = lane & 1;
        float r = (odd ? y[1] : y[0]) + dpp<DPP_XOR1>(odd ? y[0] : y[1]);
        if constexpr (P >= 4) {
            const bool high = lane & 2;
            const float t = (odd ? y[3] : y[2]) + dpp<DPP_XOR1>(odd ? y[2] : y[3]);
            r = (high ? t : r) + dpp<DPP_XOR2>(high ? r : t);
        }
        if constexpr (P >= 16) r += dpp<DPP_ROR8>(r);
        if constexpr (P >= 8) r += dpp<DPP_SHL4>(r);      // lane i += lane i + 4 (within 16; the lanes that count have a partner)
        return r;
    }
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

// A thread's part of a tile of R steps: V neighbouring channels (column `cc`) of PER rows.  V = 2: one access covers a pair, so that a
// row of 64 channels is read by 32 lanes and its staged values are written to LDS without bank conflicts.
template <int P, int V, int R>
struct Part {
    static constexpr int CH = SCAN_THREADS / P, COLS = CH / V, STEP = SCAN_THREADS / COLS, PER = R / STEP;
    static_assert(R % STEP == 0, "whole rows");
    int cc, t;
    __device__ __forceinline__ Part() : cc((threadIdx.x % COLS) * V), t(threadIdx.x / COLS) {}
    __device__ __forceinline__ int row(int i) const { return t + i * STEP; }
};

// One sample tensor as a thread sees it: uniform row addresses plus a 32-bit offset of its own (the host checks that it fits).
template <typename T, int V, typename PART>
struct Stream {
    const T* p;
    long long ts;
    unsigned off;
    __device__ __forceinline__ Stream(const void* base, long long bs, long long ts_, int b, int c0, const PART& part)
        : p(base ? (const T*)base + b * bs + c0 : nullptr), ts(ts_), off((unsigned)((part.t * (int)ts_ + part.cc) * (int)sizeof(T))) {}
    template <bool WHOLE>
    __device__ __forceinline__ void fetch(Vec<T, V> (&v)[PART::PER], const PART& part, int t0, int end, bool ok) const {
#pragma unroll
        for (int i = 0; i < PART::PER; ++i)
            if (WHOLE || (ok && t0 + part.row(i) < end))
                v[i] = *reinterpret_cast<const Vec<T, V>*>((const char*)(p + (long long)(t0 + i * PART::STEP) * ts) + off);
    }
};

// zeros to rows t0 .. end of a workgroup's columns of CH channels, `nvalid` of them there, in a result [..][D]
template <typename T, int CH, int V>
__device__ __forceinline__ void zero_rows(T* p, int D, int t0, int end, int nvalid) {
    constexpr int COLS = CH / V;
    const int cc = threadIdx.x % COLS * V;
    Vec<T, V> zero;
#pragma unroll
    for (int j = 0; j < V; ++j) zero.v[j] = (T)0.f;
    if (cc < nvalid)
        for (int t = t0 + (int)threadIdx.x / COLS; t < end; t += SCAN_THREADS / COLS) store_vec(p + (long long)t * D + cc, zero);
}

// f(true) for a tile whose steps and channels all count, f(false) otherwise
template <typename F>
__device__ __forceinline__ void whole_or_not(bool whole, F f) {
    if (whole) f(std::integral_constant<bool, true>{});
    else f(std::integral_constant<bool, false>{});
}

// delta of a thread's samples
template <typename T, int V, int PER>
__device__ __forceinline__ void deltas(float (&d)[PER][V], const Vec<T, V> (&raw)[PER], const float (&bias)[V], int with_softplus) {
#pragma unroll
    for (int i = 0; i < PER; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) d[i][j] = (float)raw[i].v[j] + bias[j];
    if (with_softplus) {
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) d[i][j] = softplus(d[i][j]);
    }
}
template <int V>
__device__ __forceinline__ void put_pairs(float2* dst, const float (&a)[V], const float (&b)[V]) {
    if constexpr (V == 2) *reinterpret_cast<float4*>(dst) = make_float4(a[0], b[0], a[1], b[1]);
    else *dst = make_float2(a[0], b[0]);
}

// rows of B or C (of this group) as fp32 into LDS, zero past the sequence and past N
template <typename T, int P, int R>
struct Shared {
    static constexpr int PER = (R * 4 * P + SCAN_THREADS - 1) / SCAN_THREADS;
    T v[PER];
    __device__ __forceinline__ void fetch(const T* p, long long ts, int N, int t0, int len) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = threadIdx.x + i * SCAN_THREADS, t = t0 + e / (4 * P), n = e % (4 * P);
            v[i] = (T)0.f;
            if (e < R * 4 * P && t < len && n < N) v[i] = p[(long long)t * ts + n];
        }
    }
    __device__ __forceinline__ void put(float (*dst)[4 * P]) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = threadIdx.x + i * SCAN_THREADS;
            if (e < R * 4 * P) (&dst[0][0])[e] = (float)v[i];
        }
    }
};

// A log2(e): rounded once more than delta A would be, by half a step of the exponent, which saves a product a state and step
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
// the same in the library's own arrays [..][4P]
__device__ __forceinline__ void load_four(const float* p, float (&x)[4]) {
    const float4 v = *reinterpret_cast<const float4*>(p);
    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void store_four(float* p, const float (&x)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}

// LDS operands of S steps
template <int P, bool SUMMARY>
struct Group {
    static constexpr int S = Steps<P>::S;
    float2 dx[S];
    float b[S][4], c[SUMMARY ? 1 : S][4];
    template <typename DX, typename B, typename C>
    __device__ __forceinline__ void read(const DX& sDX, const B& sB, const C& sC, int t, int ch, int q) {
#pragma unroll
        for (int k = 0; k < S; ++k) {
            dx[k] = sDX[t + k][ch];
            load_four(&sB[t + k][4 * q], b[k]);
            if constexpr (!SUMMARY) load_four(&sC[t + k][4 * q], c[k]);
        }
    }
};

// SUMMARY: only what the steps of a chunk do to a state: x_end = exp2(a dsum) x_begin + xin, started from zero.
// Otherwise the scan itself from the state before the chunk.
template <typename T, int P, int V, bool SUMMARY>
__global__ __launch_bounds__(SCAN_THREADS, P == 1 ? 1 : P == 2 ? 2 : 3) void scan_fwd_kernel(ScanDev s) {
    constexpr int CH = SCAN_THREADS / P, S = Steps<P>::S;
    __shared__ __attribute__((aligned(16))) float2 sDX[SCAN_T][CH];   // delta, delta u
    __shared__ __attribute__((aligned(16))) float sB[SCAN_T][4 * P], sC[SUMMARY ? 1 : SCAN_T][4 * P], sY[SUMMARY ? 1 : SCAN_T][CH];
    const nmpc_scan_args& a = s.a;
    const ScanPlace<P> at(s);
    const Part<P, V, SCAN_T> part;
    constexpr int PER = Part<P, V, SCAN_T>::PER;
    const int tid = threadIdx.x, c = tid / P, q = tid % P, ch = at.c0 + c;
    const bool ok = c < at.nvalid, mine = part.cc < at.nvalid;
    float A[4], x[4] = {0.f, 0.f, 0.f, 0.f}, total = 0.f;
    load_A<P>(s, ch, ok, q, A);
    float* chunk_state = s.xin + ((long long)(at.b * s.nch + at.chunk) * a.D + ch) * (4 * P) + 4 * q;
    if (!SUMMARY && ok) {
        if (s.nch > 1) load_four(chunk_state, x);
        else if (a.start) load_states(a.start + ((long long)at.b * a.D + ch) * a.N, a.N, q, x);
    }
    using PT = Part<P, V, SCAN_T>;
    const Stream<T, V, PT> u(a.u, a.u_bs, a.u_ts, at.b, at.c0, part), dt(a.dt, a.dt_bs, a.dt_ts, at.b, at.c0, part),
        z(SUMMARY ? nullptr : a.z, a.z_bs, a.z_ts, at.b, at.c0, part);
    const T* B = (const T*)a.B + at.b * a.B_bs + (long long)at.g * a.N;
    const T* C = (const T*)a.C + at.b * a.C_bs + (long long)at.g * a.N;
    float bias[V], skip[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = a.dt_bias && mine ? a.dt_bias[at.c0 + part.cc + j] : 0.f;
        skip[j] = !SUMMARY && a.D_skip && mine ? a.D_skip[at.c0 + part.cc + j] : 0.f;
    }
    // tiles behind the sequence are not worked on: nothing but zeros to write
    const int tile0 = at.chunk * s.tpc, tile2 = min(tile0 + s.tpc, s.ntile), tile1 = min(tile2, (at.len + SCAN_T - 1) / SCAN_T);
    auto whole = [&](int t0) { return at.nvalid == CH && t0 + SCAN_T <= at.len; };
    Vec<T, V> nd[PER], nu[PER], nz[PER], cu[PER], cz[PER];           // the next tile's samples, this one's
    Shared<T, P, SCAN_T> nB, nC;
    auto next = [&](int t0) {
        whole_or_not(whole(t0), [&](auto w) {
            dt.template fetch<w.value>(nd, part, t0, at.len, mine);
            u.template fetch<w.value>(nu, part, t0, at.len, mine);
            if (!SUMMARY && z.p) z.template fetch<w.value>(nz, part, t0, at.len, mine);
        });
        nB.fetch(B, a.B_ts, a.N, t0, at.len);
        if constexpr (!SUMMARY) nC.fetch(C, a.C_ts, a.N, t0, at.len);
    };
    if (tile0 < tile1) next(tile0 * SCAN_T);
    for (int tile = tile0; tile < tile1; ++tile) {
        const int t0 = tile * SCAN_T;
        whole_or_not(whole(t0), [&](auto w) {
            float d[PER][V];
            deltas(d, nd, bias, a.softplus);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                float du[V];
                const bool in = w.value || (mine && t0 + part.row(i) < at.len);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    du[j] = in ? d[i][j] * (float)nu[i].v[j] : 0.f;
                    d[i][j] = in ? d[i][j] : 0.f;
                }
                put_pairs<V>(&sDX[part.row(i)][part.cc], d[i], du);
                cu[i] = nu[i];
                cz[i] = nz[i];
            }
        });
        nB.put(sB);
        if constexpr (!SUMMARY) nC.put(sC);
        __syncthreads();
        if (tile + 1 < tile1) next(t0 + SCAN_T);
        // groups of S steps; the next group's operands are read from LDS while this one is computed
        Group<P, SUMMARY> cur, ahead;
        cur.read(sDX, sB, sC, 0, c, q);
#pragma unroll
        for (int t4 = 0; t4 < SCAN_T; t4 += S) {
            if (t4 + S < SCAN_T) ahead.read(sDX, sB, sC, t4 + S, c, q);
            if constexpr (!SUMMARY) {
                if (t4 % SCAN_SAVE == 0 && a.saved && ok && t0 + t4 < a.L)
                    store_four((float*)a.saved + (((long long)at.b * ((a.L + SCAN_SAVE - 1) / SCAN_SAVE) + (t0 + t4) / SCAN_SAVE) * a.D + ch) * (4 * P) + 4 * q, x);
            }
            float y[S];
#pragma unroll
            for (int k = 0; k < S; ++k) {
                const float2 dx = cur.dx[k];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_exp2f(dx.x * A[i]) * x[i] + dx.y * cur.b[k][i];
                if constexpr (SUMMARY) total += dx.x;
                else y[k] = cur.c[k][0] * x[0] + cur.c[k][1] * x[1] + cur.c[k][2] * x[2] + cur.c[k][3] * x[3];
            }
            if constexpr (!SUMMARY) {
                const float r = sum_steps<P>(y, tid);
                if (P <= 4 || q < 4) sY[t4 + (q & 3)][c] = r;
            }
            cur = ahead;
        }
        __syncthreads();
        if constexpr (!SUMMARY) {
            T* y = (T*)a.y + ((long long)at.b * a.L + t0) * a.D + at.c0;
            whole_or_not(whole(t0), [&](auto w) {
#pragma unroll
                for (int i = 0; i < PER; ++i) {
                    const int t = part.row(i);
                    if (!w.value && (!mine || t0 + t >= a.L)) continue;
                    const bool in = w.value || t0 + t < at.len;
                    Vec<T, V> o;
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        float v = sY[t][part.cc + j] + skip[j] * (float)cu[i].v[j];
                        if (z.p) {
                            const float zz = (float)cz[i].v[j];
                            v *= zz * sigmoid(zz);
                        }
                        o.v[j] = (T)(in ? v : 0.f);
                    }
                    store_vec(y + (long long)(i * PT::STEP) * a.D + (unsigned)(part.t * a.D + part.cc), o);
                }
            });
        }
    }
    if constexpr (!SUMMARY)
        zero_rows<T, CH, V>((T*)a.y + (long long)at.b * a.L * a.D + at.c0, a.D, max(tile0, tile1) * SCAN_T, min(tile2 * SCAN_T, a.L), at.nvalid);
    if (!ok) return;
    if constexpr (SUMMARY) {
        store_four(chunk_state, x);
        if (q == 0) s.dsum[(long long)(at.b * s.nch + at.chunk) * a.D + ch] = total;
    } else if (a.last && at.chunk == s.nch - 1) {
        store_states(a.last + ((long long)at.b * a.D + ch) * a.N, a.N, q, x);
    }
}

// The scan with the time axis cut inside a workgroup: each of its four waves owns 16 of 64 steps of the same 64 / P channels.  A wave
// first scans its steps from zero, keeping their decays in registers, the waves trade end states and total decays through LDS, and
// each scans again from the state it now knows - without the exponentials: 8.5 instead of 6.5 slots a state and step, but no pass over
// the samples before.  All staging is the wave's own; one barrier per 64 steps.
template <typename T, int P, int V>
__global__ __launch_bounds__(SCAN_THREADS, P == 1 ? 1 : 2) void scan_slots_kernel(ScanDev s) {
    constexpr int CH = 64 / P, S = Steps<P>::S, R = SCAN_SAVE, SLOTS = 4;
    constexpr int COLS = CH / V, STEP = 64 / COLS, PER = R / STEP, NB = R * 4 * P / 64;
    static_assert(R % STEP == 0 && 64 % COLS == 0, "whole rows");
    __shared__ __attribute__((aligned(16))) float2 sDX[SLOTS][R][CH];
    __shared__ __attribute__((aligned(16))) float sB[SLOTS][R][4 * P], sC[SLOTS][R][4 * P], sY[SLOTS][R][CH];
    __shared__ __attribute__((aligned(16))) float ends[2][SLOTS][64][8];     // end state and total decay of every lane, in turn
    const nmpc_scan_args& a = s.a;
    // workgroups go to the 8 dies in turn: neighbouring channels, which share cache lines, go to the same one
    const int nblk = (s.per + CH - 1) / CH, nx = a.G * nblk, total = a.nb * nx;
    int id = blockIdx.x;
    {
        const int xcd = id & 7, k = id >> 3, q8 = total >> 3, r8 = total & 7;
        id = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + k;
    }
    const int b = id / nx, g = id % nx / nblk, first = id % nx % nblk * CH, c0 = g * s.per + first, nvalid = min(CH, s.per - first);
    const int len = seq_length(a.lengths, b, a.L);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane / P, q = lane % P, ch = c0 + c;
    const int cc = lane % COLS * V, row0 = lane / COLS;
    const bool ok = c < nvalid, mine = cc < nvalid;
    float A[4], carry[4] = {0.f, 0.f, 0.f, 0.f};
    load_A<P>(s, ch, ok, q, A);
    if (ok && a.start) load_states(a.start + ((long long)b * a.D + ch) * a.N, a.N, q, carry);
    const T* u = (const T*)a.u + b * a.u_bs + c0 + cc;
    const T* dt = (const T*)a.dt + b * a.dt_bs + c0 + cc;
    const T* z = a.z ? (const T*)a.z + b * a.z_bs + c0 + cc : nullptr;
    const T* B = (const T*)a.B + b * a.B_bs + (long long)g * a.N;
    const T* C = (const T*)a.C + b * a.C_bs + (long long)g * a.N;
    float bias[V], skip[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = a.dt_bias && mine ? a.dt_bias[c0 + cc + j] : 0.f;
        skip[j] = a.D_skip && mine ? a.D_skip[c0 + cc + j] : 0.f;
    }
    Vec<T, V> nd[PER], nu[PER], nz[PER], cu[PER], cz[PER];
    T nB[NB], nC[NB];
    auto next = [&](int t0) {                         // this wave's 16 steps from t0 on
        whole_or_not(nvalid == CH && t0 + R <= len, [&](auto whole) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int t = t0 + row0 + i * STEP;
                if (whole.value || (mine && t < len)) {
                    nd[i] = load_vec<T, V>(dt + (long long)t * a.dt_ts);
                    nu[i] = load_vec<T, V>(u + (long long)t * a.u_ts);
                    if (z) nz[i] = load_vec<T, V>(z + (long long)t * a.z_ts);
                }
            }
        });
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int e = lane + i * 64, t = t0 + e / (4 * P), n = e % (4 * P);
            const bool in = t < len && n < a.N;
            nB[i] = in ? B[(long long)t * a.B_ts + n] : (T)0.f;
            nC[i] = in ? C[(long long)t * a.C_ts + n] : (T)0.f;
        }
    };
    next(w * R);
    const int tiles = (len + SLOTS * R - 1) / (SLOTS * R);    // behind the sequence there is nothing but zeros to write
    for (int tile = 0; tile < tiles; ++tile) {
        const int t0 = (tile * SLOTS + w) * R;
        whole_or_not(nvalid == CH && t0 + R <= len, [&](auto whole) {
            float d[PER][V];
            deltas(d, nd, bias, a.softplus);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                float du[V];
                const bool in = whole.value || (mine && t0 + row0 + i * STEP < len);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    du[j] = in ? d[i][j] * (float)nu[i].v[j] : 0.f;
                    d[i][j] = in ? d[i][j] : 0.f;
                }
                put_pairs<V>(&sDX[w][row0 + i * STEP][cc], d[i], du);
                cu[i] = nu[i];
                cz[i] = nz[i];
            }
        });
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            (&sB[w][0][0])[lane + i * 64] = (float)nB[i];
            (&sC[w][0][0])[lane + i * 64] = (float)nC[i];
        }
        __builtin_amdgcn_wave_barrier();              // the wave's own LDS operations are served in order
        next(t0 + SLOTS * R);
        float es[R][4], x[4] = {0.f, 0.f, 0.f, 0.f}, total_d = 0.f;
#pragma unroll
        for (int t = 0; t < R; ++t) {
            const float2 dx = sDX[w][t][c];
            float b4[4];
            load_four(&sB[w][t][4 * q], b4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                es[t][i] = __builtin_amdgcn_exp2f(dx.x * A[i]);
                x[i] = es[t][i] * x[i] + dx.y * b4[i];
            }
            total_d += dx.x;
        }
        float (*end)[64][8] = ends[tile & 1];
        store_four(end[w][lane], x);
        {
            float root[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) root[i] = growth_root(total_d * A[i]);
            store_four(end[w][lane] + 4, root);
        }
        __syncthreads();                              // (the other half of `ends` is free again: everyone is past its reads)
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
            float xe[4], root[4];
            load_four(end[k][lane], xe);
            load_four(end[k][lane] + 4, root);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = k == w ? carry[i] : x[i];
                carry[i] = root[i] * (root[i] * (root[i] * carry[i])) + xe[i];
            }
        }
        if (a.saved && ok && t0 < a.L)
            store_four((float*)a.saved + (((long long)b * ((a.L + R - 1) / R) + t0 / R) * a.D + ch) * (4 * P) + 4 * q, x);
#pragma unroll
        for (int t4 = 0; t4 < R; t4 += S) {
            float y[S];
#pragma unroll
            for (int k = 0; k < S; ++k) {
                const int t = t4 + k;
                const float dx = sDX[w][t][c].y;
                float b4[4], c4[4];
                load_four(&sB[w][t][4 * q], b4);
                load_four(&sC[w][t][4 * q], c4);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = es[t][i] * x[i] + dx * b4[i];
                y[k] = c4[0] * x[0] + c4[1] * x[1] + c4[2] * x[2] + c4[3] * x[3];
            }
            const float r = sum_steps<P>(y, lane);
            if (P <= 4 || q < 4) sY[w][t4 + (q & 3)][c] = r;
        }
        __builtin_amdgcn_wave_barrier();
        T* yo = (T*)a.y + ((long long)b * a.L + t0) * a.D + c0 + cc;
        whole_or_not(nvalid == CH && t0 + R <= len, [&](auto whole) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int t = row0 + i * STEP;
                if (!whole.value && (!mine || t0 + t >= a.L)) continue;
                const bool in = whole.value || t0 + t < len;
                Vec<T, V> o;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float v = sY[w][t][cc + j] + skip[j] * (float)cu[i].v[j];
                    if (z) {
                        const float zz = (float)cz[i].v[j];
                        v *= zz * sigmoid(zz);
                    }
                    o.v[j] = (T)(in ? v : 0.f);
                }
                store_vec(yo + (long long)t * a.D, o);
            }
        });
    }
    zero_rows<T, CH, V>((T*)a.y + (long long)b * a.L * a.D + c0, a.D, tiles * SLOTS * R, a.L, nvalid);
    if (ok && a.last && w == 0) store_states(a.last + ((long long)b * a.D + ch) * a.N, a.N, q, carry);
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
        const float root = growth_root(A * s.dsum[at * a.D + ch]);
        x = root * (root * (root * x)) + own;
    }
}

// The adjoint's summary of a chunk: lam before its first step, times that step's decay, started from zero behind its last.
template <typename T, int P, int V>
__global__ __launch_bounds__(SCAN_THREADS) void scan_bwd_summary_kernel(ScanDev s) {
    constexpr int CH = SCAN_THREADS / P;
    __shared__ __attribute__((aligned(16))) float2 sDG[SCAN_T][CH];   // delta, g
    __shared__ __attribute__((aligned(16))) float sC[SCAN_T][4 * P];
    const nmpc_scan_args& a = s.a;
    const ScanPlace<P> at(s);
    const Part<P, V, SCAN_T> part;
    constexpr int PER = Part<P, V, SCAN_T>::PER;
    const int tid = threadIdx.x, c = tid / P, q = tid % P, ch = at.c0 + c;
    const bool ok = c < at.nvalid, mine = part.cc < at.nvalid;
    float A[4], lam[4] = {0.f, 0.f, 0.f, 0.f}, total = 0.f, bias[V];
    load_A<P>(s, ch, ok, q, A);
#pragma unroll
    for (int j = 0; j < V; ++j) bias[j] = a.dt_bias && mine ? a.dt_bias[at.c0 + part.cc + j] : 0.f;
    using PT = Part<P, V, SCAN_T>;
    const Stream<T, V, PT> dt(a.dt, a.dt_bs, a.dt_ts, at.b, at.c0, part), z(a.z, a.z_bs, a.z_ts, at.b, at.c0, part),
        dy(a.dy, a.dy_bs, a.dy_ts, at.b, at.c0, part);
    const T* C = (const T*)a.C + at.b * a.C_bs + (long long)at.g * a.N;
    const int tile0 = at.chunk * s.tpc, tile1 = min(min(tile0 + s.tpc, s.ntile), (at.len + SCAN_T - 1) / SCAN_T);
    auto whole = [&](int t0) { return at.nvalid == CH && t0 + SCAN_T <= at.len; };
    Vec<T, V> nd[PER], ng[PER], nz[PER];
    Shared<T, P, SCAN_T> nC;
    auto next = [&](int t0) {
        whole_or_not(whole(t0), [&](auto w) {
            dt.template fetch<w.value>(nd, part, t0, at.len, mine);
            dy.template fetch<w.value>(ng, part, t0, at.len, mine);
            if (z.p) z.template fetch<w.value>(nz, part, t0, at.len, mine);
        });
        nC.fetch(C, a.C_ts, a.N, t0, at.len);
    };
    if (tile0 < tile1) next((tile1 - 1) * SCAN_T);
    for (int tile = tile1 - 1; tile >= tile0; --tile) {
        const int t0 = tile * SCAN_T;
        whole_or_not(whole(t0), [&](auto w) {
            float d[PER][V];
            deltas(d, nd, bias, a.softplus);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                float g[V];
                const bool in = w.value || (mine && t0 + part.row(i) < at.len);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    g[j] = (float)ng[i].v[j];
                    if (z.p) {
                        const float zz = (float)nz[i].v[j];
                        g[j] *= zz * sigmoid(zz);
                    }
                    g[j] = in ? g[j] : 0.f;
                    d[i][j] = in ? d[i][j] : 0.f;
                }
                put_pairs<V>(&sDG[part.row(i)][part.cc], d[i], g);
            }
        });
        nC.put(sC);
        __syncthreads();
        if (tile > tile0) next(t0 - SCAN_T);
#pragma unroll 4
        for (int t = SCAN_T - 1; t >= 0; --t) {
            const float2 dg = sDG[t][c];
            float C4[4];
            load_four(&sC[t][4 * q], C4);
#pragma unroll
            for (int i = 0; i < 4; ++i) lam[i] = (lam[i] + C4[i] * dg.y) * __builtin_amdgcn_exp2f(dg.x * A[i]);
            total += dg.x;
        }
        __syncthreads();
    }
    if (!ok) return;
    store_four(s.xin + ((long long)(at.b * s.nch + at.chunk) * a.D + ch) * (4 * P) + 4 * q, lam);
    if (q == 0) s.dsum[(long long)(at.b * s.nch + at.chunk) * a.D + ch] = total;
}

// Sums over a wave's 64 / P channels of the eight values dB[4], dC[4] of every lane.  Lanes trade halves as in sum_steps: after the
// exchanges across 32, 16 and 8 lanes a lane holds the one value 4 (lane >> 5) + 2 (lane >> 4 & 1) + (lane >> 3 & 1) of its states 4q ..,
// and the channels that are left (fewer than 8 lanes apart) are added up.  dst: the wave's row [2][4P] of this step.
__device__ __forceinline__ float trade32(float x, float y) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
    const unsigned a = r[0], b = r[1];                // (a bit cast of r[1] itself would read r[0])
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float trade16(float x, float y) {
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, y), false, false);
    const unsigned a = r[0], b = r[1];                // (a bit cast of r[1] itself would read r[0])
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}
template <int P>
__device__ __forceinline__ void sum_channels(const float (&p)[8], int lane, int q, float* dst) {
    float v[4], w[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = trade32(p[i], p[4 + i]);
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = trade16(v[i], v[2 + i]);
    const int n = 4 * q + 2 * (lane >> 4 & 1);
    float* out = dst + (lane >> 5) * (4 * P);
    if constexpr (P == 16) {
        out[n] = w[0];
        out[n + 1] = w[1];
    } else {
        const bool hi = lane & 8;
        float r = (hi ? w[1] : w[0]) + dpp<DPP_ROR8>(hi ? w[0] : w[1]);
        if constexpr (P <= 4) r += dpp<DPP_SHL4>(r);
        if constexpr (P <= 2) r += dpp<DPP_XOR2>(r);
        if constexpr (P == 1) r += dpp<DPP_XOR1>(r);
        if (P == 8 || (lane & 7) < P) out[n + (lane >> 3 & 1)] = r;
    }
}

// Tiles of 16 steps from the last to the first: the states and decays of a tile are recomputed from the state saved before it and
// stay in registers, then the adjoint runs back through them.
template <typename T, int P, int V>
__global__ __launch_bounds__(SCAN_THREADS, P == 1 ? 1 : 2) void scan_bwd_kernel(ScanDev s) {
    constexpr int CH = SCAN_THREADS / P, NP = 4 * P, R = SCAN_SAVE, S = Steps<P>::S;
    __shared__ __attribute__((aligned(16))) float2 sDU[R][CH], sS[R][CH];   // delta, u;  sum_n lam B, sum_n lam h A log2(e)
    __shared__ __attribute__((aligned(16))) float sG[R][CH], sY[R][CH], sB[R][NP], sC[R][NP];
    __shared__ float sP[4][R][2 * NP];                // each wave's sums of dB, dC over its channels
    const nmpc_scan_args& a = s.a;
    const ScanPlace<P> at(s);
    const Part<P, V, R> part;
    constexpr int PER = Part<P, V, R>::PER;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = tid / P, q = tid % P, ch = at.c0 + c;
    const bool ok = c < at.nvalid, mine = part.cc < at.nvalid;
    float A[4], lam[4] = {0.f, 0.f, 0.f, 0.f}, dA[4] = {0.f, 0.f, 0.f, 0.f}, dD[2] = {0.f, 0.f}, db[2] = {0.f, 0.f}, bias[V], skip[V];
    load_A<P>(s, ch, ok, q, A);
    const long long row = (long long)at.b * s.nch + at.chunk;
    if (ok) {
        if (s.nch > 1) load_four(s.xin + (row * a.D + ch) * NP + 4 * q, lam);
        else if (a.dlast) load_states(a.dlast + ((long long)at.b * a.D + ch) * a.N, a.N, q, lam);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        bias[j] = a.dt_bias && mine ? a.dt_bias[at.c0 + part.cc + j] : 0.f;
        skip[j] = a.D_skip && mine ? a.D_skip[at.c0 + part.cc + j] : 0.f;
    }
    using PT = Part<P, V, R>;
    const Stream<T, V, PT> u(a.u, a.u_bs, a.u_ts, at.b, at.c0, part), dt(a.dt, a.dt_bs, a.dt_ts, at.b, at.c0, part),
        z(a.z, a.z_bs, a.z_ts, at.b, at.c0, part), dy(a.dy, a.dy_bs, a.dy_ts, at.b, at.c0, part);
    const T* B = (const T*)a.B + at.b * a.B_bs + (long long)at.g * a.N;
    const T* C = (const T*)a.C + at.b * a.C_bs + (long long)at.g * a.N;
    auto whole = [&](int t0) { return at.nvalid == CH && t0 + R <= at.len; };
    const int ntile = (a.L + R - 1) / R, tile0 = at.chunk * s.tpc * (SCAN_T / R), tile2 = min(tile0 + s.tpc * (SCAN_T / R), ntile);
    const int tile1 = min(tile2, (at.len + R - 1) / R);       // tiles behind the sequence: zeros; their sums are not read
    {
        const long long seq = (long long)at.b * a.L * a.D + at.c0;
        const int t0 = max(tile0, tile1) * R, end = min(tile2 * R, a.L);
        zero_rows<T, CH, V>((T*)a.du + seq, a.D, t0, end, at.nvalid);
        zero_rows<T, CH, V>((T*)a.ddt + seq, a.D, t0, end, at.nvalid);
        if (a.z) zero_rows<T, CH, V>((T*)a.dz + seq, a.D, t0, end, at.nvalid);
    }
    Vec<T, V> nd[PER], nu[PER], ng[PER], nz[PER], cd[PER], cg[PER], cz[PER];
    Shared<T, P, R> nB, nC;
    auto next = [&](int t0) {
        whole_or_not(whole(t0), [&](auto w) {
            dt.template fetch<w.value>(nd, part, t0, at.len, mine);
            u.template fetch<w.value>(nu, part, t0, at.len, mine);
            dy.template fetch<w.value>(ng, part, t0, at.len, mine);
            if (z.p) z.template fetch<w.value>(nz, part, t0, at.len, mine);
        });
        nB.fetch(B, a.B_ts, a.N, t0, at.len);
        nC.fetch(C, a.C_ts, a.N, t0, at.len);
    };
    if (tile0 < tile1) next((tile1 - 1) * R);
    for (int tile = tile1 - 1; tile >= tile0; --tile) {
        const int t0 = tile * R;
        float x0[4] = {0.f, 0.f, 0.f, 0.f}, xs[R][4], es[R][4];
        if (ok) load_four((const float*)a.saved + (((long long)at.b * ntile + tile) * a.D + ch) * NP + 4 * q, x0);
        whole_or_not(whole(t0), [&](auto w) {
            float d[PER][V];
            deltas(d, nd, bias, a.softplus);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const bool in = w.value || (mine && t0 + part.row(i) < at.len);
                float uu[V];
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float g = (float)ng[i].v[j];
                    if (z.p) {
                        const float zz = (float)nz[i].v[j];
                        g *= zz * sigmoid(zz);
                    }
                    uu[j] = in ? (float)nu[i].v[j] : 0.f;
                    d[i][j] = in ? d[i][j] : 0.f;
                    sG[part.row(i)][part.cc + j] = in ? g : 0.f;
                }
                put_pairs<V>(&sDU[part.row(i)][part.cc], d[i], uu);
                cd[i] = nd[i]; cg[i] = ng[i]; cz[i] = nz[i];
            }
        });
        nB.put(sB);
        nC.put(sC);
        __syncthreads();
        if (tile > tile0) next(t0 - R);
#pragma unroll
        for (int t4 = 0; t4 < R; t4 += S) {
            float y[S];
#pragma unroll
            for (int k = 0; k < S; ++k) {
                const int t = t4 + k;
                const float2 du = sDU[t][c];
                const float w = du.x * du.y;
                float b[4];
                load_four(&sB[t][4 * q], b);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    es[t][i] = __builtin_amdgcn_exp2f(du.x * A[i]);
                    xs[t][i] = es[t][i] * (t ? xs[t ? t - 1 : 0][i] : x0[i]) + w * b[i];
                }
                if (z.p) {
                    float C4[4];
                    load_four(&sC[t][4 * q], C4);
                    y[k] = C4[0] * xs[t][0] + C4[1] * xs[t][1] + C4[2] * xs[t][2] + C4[3] * xs[t][3];
                }
            }
            if (z.p) {
                const float r = sum_steps<P>(y, tid);
                if (P <= 4 || q < 4) sY[t4 + (q & 3)][c] = r;
            }
        }
#pragma unroll
        for (int t4 = R - S; t4 >= 0; t4 -= S) {
            float s1[S], s2[S];
#pragma unroll
            for (int k = S - 1; k >= 0; --k) {
                const int t = t4 + k;
                const float2 du = sDU[t][c];
                const float g = sG[t][c], w = du.x * du.y;
                float b[4], C4[4], p[8];
                load_four(&sB[t][4 * q], b);
                load_four(&sC[t][4 * q], C4);
                s1[k] = s2[k] = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    lam[i] += C4[i] * g;
                    p[i] = lam[i] * w;
                    p[4 + i] = xs[t][i] * g;
                    s1[k] += lam[i] * b[i];
                    lam[i] *= es[t][i];
                    const float m = lam[i] * (t ? xs[t ? t - 1 : 0][i] : x0[i]);
                    s2[k] += m * A[i];
                    dA[i] += m * du.x;
                }
                sum_channels<P>(p, lane, q, sP[wave][t]);
            }
            const float r1 = sum_steps<P>(s1, tid), r2 = sum_steps<P>(s2, tid);
            if (P <= 4 || q < 4) sS[t4 + (q & 3)][c] = make_float2(r1, r2);
        }
        __syncthreads();
        const long long blk = (at.c0 - at.g * s.per) / CH;
        for (int e = tid; e < R * 2 * NP; e += SCAN_THREADS) {
            const int t = e / (2 * NP), n = e % (2 * NP);
            if (t0 + t < a.L)
                s.pBC[(((blk * a.nb + at.b) * a.L + t0 + t) * a.G + at.g) * (2 * NP) + n] = (sP[0][t][n] + sP[1][t][n]) + (sP[2][t][n] + sP[3][t][n]);
        }
        const long long out = ((long long)at.b * a.L + t0) * a.D + at.c0;
        whole_or_not(whole(t0), [&](auto w) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int t = part.row(i);
                if (!w.value && (!mine || t0 + t >= a.L)) continue;
                const bool in = w.value || t0 + t < at.len;
                Vec<T, V> ou, od, oz;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float2 sums = sS[t][part.cc + j], du = sDU[t][part.cc + j];      // zero past the sequence, as is g
                    const float g = sG[t][part.cc + j];
                    const float vu = skip[j] * g + du.x * sums.x;
                    float vd = sums.y * (1.f / LOG2E) + du.y * sums.x, vz = 0.f;
                    if (a.softplus) vd *= sigmoid((float)cd[i].v[j] + bias[j]);
                    if (z.p) {
                        const float zz = (float)cz[i].v[j], p = sigmoid(zz);
                        vz = (float)cg[i].v[j] * (sY[t][part.cc + j] + skip[j] * du.y) * (p * (1.f + zz * (1.f - p)));
                    }
                    ou.v[j] = (T)(in ? vu : 0.f); od.v[j] = (T)(in ? vd : 0.f); oz.v[j] = (T)(in ? vz : 0.f);
                    if (in) {
                        dD[V == 2 ? j : i & 1] += g * du.y;
                        db[V == 2 ? j : i & 1] += vd;
                    }
                }
                const long long o = out + (long long)(i * PT::STEP) * a.D + (unsigned)(part.t * a.D + part.cc);
                store_vec((T*)a.du + o, ou);
                store_vec((T*)a.ddt + o, od);
                if (z.p) store_vec((T*)a.dz + o, oz);
            }
        });
        __syncthreads();                              // sG, sDU and sP are written again
    }
    if (ok) {
        store_four(s.pA + (row * a.D + ch) * NP + 4 * q, dA);
        if (a.dstart && at.chunk == 0) store_states(a.dstart + ((long long)at.b * a.D + ch) * a.N, a.N, q, lam);
    }
    // dD and the bias, joined over the threads that share channels.  A thread has two sums each: of two channels (V = 2), or of its even
    // and odd rows (V = 1), so that the order of additions, and with it the result, is the same for both.
    constexpr int COLS = Part<P, V, R>::COLS, STEP = Part<P, V, R>::STEP, CLASSES = V == 2 || PER == 1 ? STEP : 2 * STEP;
    float* red = &sDU[0][0].x;
    static_assert(sizeof(sDU) >= 4 * SCAN_THREADS * sizeof(float) || (V == 1 && PER == 1), "reduction buffer");
#pragma unroll
    for (int j = 0; j < (V == 2 || PER > 1 ? 2 : 1); ++j) {
        red[(2 * j) * SCAN_THREADS + tid] = dD[j];
        red[(2 * j + 1) * SCAN_THREADS + tid] = db[j];
    }
    __syncthreads();
    if (tid < at.nvalid) {
        float v0 = 0.f, v1 = 0.f;
        for (int k = 0; k < CLASSES; ++k) {
            const int j = V == 2 ? tid & 1 : k / STEP, r = (V == 2 ? k : k % STEP) * COLS + tid / V;
            v0 += red[(2 * j) * SCAN_THREADS + r];
            v1 += red[(2 * j + 1) * SCAN_THREADS + r];
        }
        s.pDb[(row * 2) * a.D + at.c0 + tid] = v0;
        s.pDb[(row * 2 + 1) * a.D + at.c0 + tid] = v1;
    }
}

// Sums of the partial sums over sequences and chunks (dA, dD, the bias) and over channel blocks (dB, dC), in a fixed order: four
// threads share a parameter's rows, each with four sums of its own, so that the loads of many rows are in flight.
__global__ __launch_bounds__(256) void scan_reduce_params_kernel(ScanDev s, int NP) {
    __shared__ float red[256];
    const nmpc_scan_args& a = s.a;
    const long long rows = (long long)a.nb * s.nch, id = (long long)blockIdx.x * 64 + (threadIdx.x & 63), nA = (long long)a.D * NP;
    const int sub = threadIdx.x >> 6;
    const bool is_A = id < nA, is_b = !is_A && id < nA + 2 * a.D;
    const float* p = is_A ? s.pA + id : s.pDb + (id - nA);
    const long long step = is_A ? nA : 2 * a.D;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (is_A || is_b)
        for (long long r = sub; r < rows; r += 16)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (r + 4 * k < rows) v[k] += p[(r + 4 * k) * step];
    red[threadIdx.x] = (v[0] + v[1]) + (v[2] + v[3]);
    __syncthreads();
    if (sub) return;
    const float sum = (red[threadIdx.x] + red[threadIdx.x + 64]) + (red[threadIdx.x + 128] + red[threadIdx.x + 192]);
    if (is_A) {
        const int n = (int)(id % NP);
        if (n < a.N) a.dA[(id / NP) * a.N + n] = sum;
    } else if (is_b) {
        const int k = (int)((id - nA) / a.D);
        float* out = k ? a.ddt_bias : a.dD;
        if (out) out[(id - nA) % a.D] = sum;
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
        const long long bt = r / a.G;
        const bool in = !a.lengths || (int)(bt % a.L) < seq_length(a.lengths, (int)(bt / a.L), a.L);
        for (int k = 0; in && k < s.nblk; ++k) v += s.pBC[(k * rows + r) * (2 * NP) + n];
        if (n < a.N) ((T*)a.dB)[r * a.N + n] = (T)v;
        else if (n >= NP && n - NP < a.N) ((T*)a.dC)[r * a.N + n - NP] = (T)v;
    }
}

// One step of every sequence; the state a.last is read and replaced: 8 N bytes a channel, which is the time.  FOUR: N is a multiple
// of 4 and a lane's four states, decays, B and C are one access each.
template <typename T, int P, bool FOUR>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanDev s) {
    const nmpc_scan_args& a = s.a;
    const unsigned id = blockIdx.x * 256u + threadIdx.x, bc = id / P;
    const int q = (int)(id % P), b = (int)(bc / (unsigned)a.D), ch = (int)(bc % (unsigned)a.D);
    if (b >= a.nb) return;                            // the P lanes of a channel leave together
    const int n0 = 4 * q;
    const long long g = (long long)(ch / s.per) * a.N + n0;
    const T* Bp = (const T*)a.B + b * a.B_bs + g;
    const T* Cp = (const T*)a.C + b * a.C_bs + g;
    const float* Ap = a.A + (long long)ch * a.N + n0;
    float* state = a.last + (long long)bc * a.N + n0;
    float A[4], x[4], B[4], C[4];
    if (FOUR) {
        if (n0 < a.N) {
            load_four(Ap, A);
            load_four(state, x);
            const Vec<T, 4> vb = load_vec<T, 4>(Bp), vc = load_vec<T, 4>(Cp);
#pragma unroll
            for (int i = 0; i < 4; ++i) { B[i] = (float)vb.v[i]; C[i] = (float)vc.v[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) A[i] = x[i] = B[i] = C[i] = 0.f;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = n0 + i < a.N;
            A[i] = in ? Ap[i] : 0.f;
            x[i] = in ? state[i] : 0.f;
            B[i] = in ? (float)Bp[i] : 0.f;
            C[i] = in ? (float)Cp[i] : 0.f;
        }
    }
    const float uu = (float)((const T*)a.u)[b * a.u_bs + ch];
    float d = (float)((const T*)a.dt)[b * a.dt_bs + ch] + (a.dt_bias ? a.dt_bias[ch] : 0.f);
    const float zz = a.z ? (float)((const T*)a.z)[b * a.z_bs + ch] : 0.f;
    if (a.softplus) d = softplus(d);
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = __builtin_amdgcn_exp2f(d * (A[i] * LOG2E)) * x[i] + (d * uu) * B[i];
        y += C[i] * x[i];
    }
    if (FOUR) {
        if (n0 < a.N) store_four(state, x);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n0 + i < a.N) state[i] = x[i];
    }
    y = sum_lanes<P>(y);
    if (q == 0) {
        if (a.D_skip) y += a.D_skip[ch] * uu;
        if (a.z) y *= zz * sigmoid(zz);
        ((T*)a.y)[bc] = (T)y;
    }
}

static int scan_lanes(int N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// How a pass runs: whole sequences one tile after the other, the time axis in slots of a workgroup (forward only), or in chunks with a
// summary pass before; the least of the estimated times (us).  Each is made of the steps that follow one another and of the work at the rate
// of a full chip (bf16, 16 states); chunks pay besides for two more launches, partial sums, and a join that goes through them one after the
// other: few channels in as many chunks as fill the chip would spend their time there, so that longer ones are looked at too.
// Measured, in us (16 states and bf16 unless noted; chunks of .. tiles):       whole   slots   chunks
//   forward   1 x 8192 x 2048 channels (268 M states and steps)                 870     350    141 (8), 150 (16), 206 (1)
//             1 x 8192 x 64                                                     870     350     85 (1),  49 (4),   64 (8)
//             1 x 2000 x 512, 8 states                                          260     101     36 (1),  33 (2),   42 (4)
//             2 x 2048 x 2048                                                   223      93     77 (4),  80 (8)
//             4 x 2048 x 2048                                                   224     116    130 (4), 134 (8)
//             8 x 2048 x 2048                                                   225     205    236 (4), 251 (16)
//             16 x 512 x 2048                                                    84      97    127 (4)
//   backward  1 x 8192 x 64                                                    3000            121 (1),  91 (2),   98 (4)
//             4 x 2048 x 2048                                                   783            320 (4), 318 (8)
//             16 x 512 x 2048                                                   252            316 (4), 362 (1)
//             64 x 100 x 256                                                     60              77 (1)
//             fp32, 64 sequences of 33 .. 64 steps, 32 .. 256 channels,
//             8 or 16 states                                                  37..46          45..50 (1)
//             the same of 100 steps, 32 .. 128 channels                       57..69          52..61 (1)
static void scan_plan(ScanDev& s, bool backward) {
    const nmpc_scan_args& a = s.a;
    const int P = scan_lanes(a.N), CH = SCAN_THREADS / P;
    s.per = a.D / a.G;
    s.nblk = (s.per + CH - 1) / CH;
    s.ntile = a.L > 0 ? (a.L + SCAN_T - 1) / SCAN_T : 0;
    s.nch = 1;
    s.tpc = s.ntile;
    s.slots = 0;
    const long long base = (long long)a.nb * a.G * s.nblk;
    if (base == 0 || s.ntile == 0) return;
    const double work = (double)a.nb * a.D * a.L * 4 * P * 1e-6;
    const double whole = std::max((backward ? 13.7 : 4.0) * s.ntile, (backward ? 1.03 : 0.35) * work);
    const double slots = backward ? 1e30 : std::max(3.0 * ((a.L + 63) / 64), 0.45 * work);
    const long long want = (1024 + base - 1) / base;            // chunks of 1024 workgroups: four a CU, of which one to three run at once
    double chunks = 1e30;
    int tpc = s.ntile;
    for (long long t = want < s.ntile ? (s.ntile + want - 1) / want : 1; t < s.ntile; t *= 2) {
        // the longer of both, and more where they are alike: workgroups that share a CU slow each other down
        const double chain = (backward ? 14.3 : 5.6) * t, bulk = (backward ? 1.10 : 0.44) * work;
        const double us = std::cbrt(chain * chain * chain + bulk * bulk * bulk) + (backward ? 24.0 : 10.0) +
                          (backward ? 0.35 : 0.26) * (double)((s.ntile + t - 1) / t);
        if (us < chunks) { chunks = us; tpc = (int)t; }
    }
    if (slots < whole && slots <= chunks) {
        s.slots = 1;
    } else if (chunks < whole) {
        s.tpc = tpc;
        s.nch = (s.ntile + tpc - 1) / tpc;
    }
}

// may the samples be accessed in pairs of channels?
template <typename T>
static bool scan_pairs(const ScanDev& s) {
    const nmpc_scan_args& a = s.a;
    return s.per % 2 == 0 && vec_ok<T>(a.u, a.u_bs, a.u_ts, 2) && vec_ok<T>(a.dt, a.dt_bs, a.dt_ts, 2) && vec_ok<T>(a.z, a.z_bs, a.z_ts, 2);
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

// the number of workgroups of a pass, 0 if a launch cannot have them
static unsigned scan_grid(const ScanDev& s) {
    const int CH = (s.slots ? 64 : SCAN_THREADS) / scan_lanes(s.a.N);
    const long long blocks = (long long)s.a.nb * (s.slots ? 1 : s.nch) * s.a.G * ((s.per + CH - 1) / CH);
    return blocks < (1 << 24) ? (unsigned)blocks : 0;
}

static int scan_check(const char* what, const nmpc_scan_args* a) {
    NMPC_REQUIRE(a, "%s: null argument", what);
    NMPC_REQUIRE(a->struct_size == (int)sizeof(nmpc_scan_args), "%s: struct of %d bytes, the library's has %d", what, a->struct_size,
                 (int)sizeof(nmpc_scan_args));
    NMPC_REQUIRE(a->dtype >= NMPC_F32 && a->dtype <= NMPC_F16, "%s: unknown element type %d", what, a->dtype);
    NMPC_REQUIRE(a->nb >= 0 && a->L >= 0 && a->D >= 1, "%s: bad sizes (%d sequences, %d steps, %d channels)", what, a->nb, a->L, a->D);
    NMPC_REQUIRE(a->L <= 1 << 30, "%s: at most 2^30 steps", what);
    NMPC_REQUIRE(a->N >= 1 && a->N <= 64, "%s: %d states a channel (1..64)", what, a->N);
    NMPC_REQUIRE(a->G >= 1 && a->D % a->G == 0, "%s: %d groups do not divide %d channels", what, a->G, a->D);
    // a launch has fewer than 2^32 threads
    NMPC_REQUIRE((long long)a->nb * a->D * 64 < (1ll << 32), "%s: too many channels for one launch", what);
    // a thread's offset within 16 rows is kept in 32 bits
    const long long most = 1ll << 24;
    auto fits = [&](const void* p, long long ts) { return !p || a->L <= 1 || (ts >= 0 && ts <= most); };
    NMPC_REQUIRE(a->D <= most && fits(a->u, a->u_ts) && fits(a->dt, a->dt_ts) && fits(a->z, a->z_ts) && fits(a->dy, a->dy_ts),
                 "%s: strides between steps of 0..2^24 elements", what);
    NMPC_REQUIRE(((uintptr_t)a->saved | (uintptr_t)a->workspace) % 16 == 0, "%s: saved and workspace start on 16 bytes", what);
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
    if (nb <= 0 || L <= 0 || L > 1 << 30 || D <= 0 || N <= 0 || N > 64) return 0;
    return (unsigned long long)nb * ((L + SCAN_SAVE - 1) / SCAN_SAVE) * D * 4 * scan_lanes(N) * sizeof(float);
}

extern "C" unsigned long long nmpc_lpv_scan_workspace_bytes(int nb, int L, int D, int N, int G, int backward) {
    if (nb <= 0 || L < 0 || L > 1 << 30 || D <= 0 || N <= 0 || N > 64 || G <= 0 || D % G) return 0;
    ScanDev s = {};
    s.a.nb = nb; s.a.L = L; s.a.D = D; s.a.N = N; s.a.G = G;
    scan_plan(s, backward != 0);
    return scan_workspace(s, backward != 0, nullptr);
}

extern "C" int nmpc_lpv_scan_plan(int nb, int L, int D, int N, int G, int backward) {
    if (nb <= 0 || L <= 0 || L > 1 << 30 || D <= 0 || N <= 0 || N > 64 || G <= 0 || D % G) return -1;
    ScanDev s = {};
    s.a.nb = nb; s.a.L = L; s.a.D = D; s.a.N = N; s.a.G = G;
    scan_plan(s, backward != 0);
    return s.slots ? 0 : s.nch;
}

extern "C" int nmpc_lpv_scan(const nmpc_scan_args* args, void* stream) {
    if (scan_check("nmpc_lpv_scan", args)) return 1;
    ScanDev s = {};
    s.a = *args;
    const nmpc_scan_args& a = s.a;
    if (a.nb == 0) return 0;
    NMPC_REQUIRE(a.A && (a.L == 0 || (a.u && a.dt && a.B && a.C && a.y)), "nmpc_lpv_scan: null argument");
    scan_plan(s, false);
    const unsigned long long need = scan_workspace(s, false, (char*)a.workspace);
    NMPC_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need), "nmpc_lpv_scan: workspace of %llu bytes, %llu needed", a.workspace_bytes, need);
    const unsigned grid = scan_grid(s);
    NMPC_REQUIRE(grid || a.nb == 0, "nmpc_lpv_scan: too many sequences and channels for one launch");
    const hipStream_t st = (hipStream_t)stream;
    NMPC_DTYPE_SWITCH(a.dtype, {
        NMPC_P_SWITCH(a.N, {
            constexpr int V_ = P_ == 16 ? 1 : 2;          // 16 channels: fewer pairs than a tile has rows for
            const bool pairs = scan_pairs<T_>(s) && vec_ok<T_>(a.y, 0, 0, 2);
            if (s.slots) {
                if (pairs) scan_slots_kernel<T_, P_, V_><<<grid, SCAN_THREADS, 0, st>>>(s);
                else scan_slots_kernel<T_, P_, 1><<<grid, SCAN_THREADS, 0, st>>>(s);
                NMPC_HIP_CHECK(hipGetLastError());
                return 0;
            }
            if (s.nch > 1) {
                if (pairs) scan_fwd_kernel<T_, P_, V_, true><<<grid, SCAN_THREADS, 0, st>>>(s);
                else scan_fwd_kernel<T_, P_, 1, true><<<grid, SCAN_THREADS, 0, st>>>(s);
                scan_chunks_kernel<false><<<(unsigned)(((long long)a.nb * a.D * 4 * P_ + 255) / 256), 256, 0, st>>>(s, 4 * P_);
            }
            if (pairs) scan_fwd_kernel<T_, P_, V_, false><<<grid, SCAN_THREADS, 0, st>>>(s);
            else scan_fwd_kernel<T_, P_, 1, false><<<grid, SCAN_THREADS, 0, st>>>(s);
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
    // the sums of the parameters' gradients: four threads a value, fewer than 2^32 a launch
    NMPC_REQUIRE((long long)a.D * (4 * scan_lanes(a.N) + 2) < 1ll << 30, "nmpc_lpv_scan_bwd: too many channels and states for one launch");
    NMPC_REQUIRE(!a.D_skip || a.dD, "nmpc_lpv_scan_bwd: D needs dD");
    NMPC_REQUIRE(!a.dt_bias || a.ddt_bias, "nmpc_lpv_scan_bwd: dt_bias needs ddt_bias");
    scan_plan(s, true);
    const unsigned long long need = a.nb > 0 ? scan_workspace(s, true, (char*)a.workspace) : 0;
    NMPC_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need), "nmpc_lpv_scan_bwd: workspace of %llu bytes, %llu needed", a.workspace_bytes, need);
    const unsigned grid = scan_grid(s);
    NMPC_REQUIRE(grid || a.nb == 0, "nmpc_lpv_scan: too many sequences and channels for one launch");
    const hipStream_t st = (hipStream_t)stream;
    NMPC_DTYPE_SWITCH(a.dtype, {
        NMPC_P_SWITCH(a.N, {
            constexpr int NP = 4 * P_, V_ = P_ == 16 ? 1 : 2;
            if (a.nb > 0) {
                const bool pairs = scan_pairs<T_>(s) && vec_ok<T_>(a.dy, a.dy_bs, a.dy_ts, 2) && vec_ok<T_>(a.du, 0, 0, 2) &&
                                   vec_ok<T_>(a.ddt, 0, 0, 2) && vec_ok<T_>(a.dz, 0, 0, 2);
                if (s.nch > 1) {
                    if (pairs) scan_bwd_summary_kernel<T_, P_, V_><<<grid, SCAN_THREADS, 0, st>>>(s);
                    else scan_bwd_summary_kernel<T_, P_, 1><<<grid, SCAN_THREADS, 0, st>>>(s);
                    scan_chunks_kernel<true><<<(unsigned)(((long long)a.nb * a.D * NP + 255) / 256), 256, 0, st>>>(s, NP);
                }
                if (pairs) scan_bwd_kernel<T_, P_, V_><<<grid, SCAN_THREADS, 0, st>>>(s);
                else scan_bwd_kernel<T_, P_, 1><<<grid, SCAN_THREADS, 0, st>>>(s);
            }
            scan_reduce_params_kernel<<<(unsigned)(((long long)a.D * (NP + 2) + 63) / 64), 256, 0, st>>>(s, NP);
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
    scan_plan(s, false);
    NMPC_DTYPE_SWITCH(a.dtype, {
        NMPC_P_SWITCH(a.N, {
            const unsigned grid = (unsigned)(((long long)a.nb * a.D * P_ + 255) / 256);
            if (a.N % 4 == 0 && vec_ok<float>(a.A, 0, 0, 4) && vec_ok<float>(a.last, 0, 0, 4) && vec_ok<T_>(a.B, a.B_bs, 0, 4) && vec_ok<T_>(a.C, a.C_bs, 0, 4))
                scan_step_kernel<T_, P_, true><<<grid, 256, 0, (hipStream_t)stream>>>(s);
            else scan_step_kernel<T_, P_, false><<<grid, 256, 0, (hipStream_t)stream>>>(s);
        })
    })
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}
