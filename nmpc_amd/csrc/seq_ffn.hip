// Gated feed-forward projections: h = act(x Wg') o (x Wu'), x[M,K], Wg / Wu[F,K], and their gradients
//   dG = dh o up o act'(gate),  dU = dh o act(gate),
//   dx = dG Wg + dU Wu,  dWg = dG' x,  dWu = dU' x.
// Both projections of a tile are accumulated side by side, so that the activation and the product happen in registers and
// neither projection is written (a training pass keeps both in fp32 for the gradient: kept in bf16 the gradients were off by 1.65
// times as much).  Products run on the matrix cores with fp32 accumulation; dG and dU are rounded to the element type once, as
// operands of the next products, which take both side by side: dx is one product over 2 F, [dWg; dWu] one of 2 F rows.
// What bounds it: many rows the matrix cores, few rows reading the weights, a prompt of a few hundred rows the latency of its loads.
// Measured: bf16 4096 x 2048 x 8192 forward 264 us (1.04 PFLOP/s), 340 with both projections kept, gradient 585 us: 0.9 PFLOP/s over
// training steps, which hold the chip at its power limit (1.83 GHz in both gradients; the library's plain products of these sizes reach
// 1.1 .. 1.3; writing the projections past the caches is 36 us faster alone and no faster in training steps); fp32 4096 x 256 x 1024
// training 162 us (80 TFLOP/s); bf16 1 x 2048 x 8192 12.9 us, 5.2 TB/s.
#include <cmath>

#include "seq_common.h"

namespace nmpc {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// value and slope of an activation
__device__ __forceinline__ float2 activation(int act, float x) {
    if (act == NMPC_ACT_TANH) {
        const float e = __builtin_amdgcn_exp2f(-2.f * LOG2E * fabsf(x)), y = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e);
        const float r = __builtin_amdgcn_rcpf(1.f + e);
        return make_float2(fabsf(x) < 0.1f ? tanhf(x) : copysignf(y, x), 4.f * e * r * r);
    }
    if (act == NMPC_ACT_GELU) {
        const float p = 0.5f * erfcf(-0.70710678f * x);
        return make_float2(x * p, p + x * 0.39894228f * __builtin_amdgcn_exp2f(-0.5f * LOG2E * x * x));
    }
    const float p = sigmoid(x), n = sigmoid(-x);
    if (act == NMPC_ACT_SIGMOID) return make_float2(p, p * n);
    return make_float2(x * p, p * (1.f + x * n));
}

// ---- products of many rows -------------------------------------------------------------------------------------------
// out[m][n] = sum_k A(m,k) B(n,k).  An operand is stored either with k contiguous (rows of whole 64-byte pieces) or with its own index
// contiguous (row k holds all m or n; up to kmax rows, a multiple of 16 bytes each).
struct NtArgs {
    const void *A, *B, *B1;            // GATED: B, B1 are the two weight matrices, side by side in n.  B stored by k: B holds k < kcut, B1 the rest
    long long a_ld, b_ld;              // elements
    int M, N, ktiles, act;
    int kcut, a_kmax, b_kmax;          // operands stored by k: rows of each part that exist (past them the other operand is zero)
    void *out, *out1;                  // rows from `cut` on go to out1 (two gradients of one product); `rows` rows of each exist
    int cut, rows;
    float* pre;                        // GATED: [2][M][N], both projections, may be null
    float* part;                       // fp32 partial products [splits][M][N] instead of out
    int splits;
    int mt, nt;                        // tiles
    int wide;                          // results may be stored in pieces of 16 bytes: rows of whole groups of eight, aligned
};

template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
    static __device__ __forceinline__ f32x16 step(uint4 a, uint4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<f16> {
    static __device__ __forceinline__ f32x16 step(uint4 a, uint4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<float> {                    // four fp32 products of depth 2: element j of both 16-byte pieces belongs to the same k
    static __device__ __forceinline__ f32x16 step(uint4 a, uint4 b, f32x16 c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
};

// eight neighbouring results, `left` of them inside the row; wide: rows are whole groups of eight
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int left, bool wide) {
    if (wide) {
        if (left <= 0) return;
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < 8; k += E) {
            Vec<T, E> o;
#pragma unroll
            for (int i = 0; i < E; ++i) o.v[i] = (T)v[k + i];
            store_vec(p + k, o);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < left) p[i] = (T)v[i];
    }
}

// 16 bytes (8 or 4 steps of k) of an operand's fragment: rows base + (lane & 31) of the tile, k pieces 2 ks + (lane >> 5)
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <typename T, int ROWS, bool KC>
struct Fragment {
    int off;                           // of this lane, for rows base ..
    __device__ __forceinline__ Fragment(int base, int lane) {
        if constexpr (KC) off = (base + (lane & 31)) * 64;
        else if constexpr (sizeof(T) == 2) {
            const int k3 = (lane >> 2) & 3;
            off = ((lane >> 5) * 8 + k3) * (ROWS * 2) + ((base / 8) ^ (k3 << 2)) * 16 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
        } else off = (lane >> 5) * 4 * (ROWS * 4) + (base + (lane & 31)) * 4;
    }
    __device__ __forceinline__ uint4 read(const char* buf, int ks, int lane) const {
        if constexpr (KC) {
            return *reinterpret_cast<const uint4*>(buf + off + ((ks * 2 + (lane >> 5)) ^ ((lane >> 2) & 3)) * 16);
        } else if constexpr (sizeof(T) == 2) {
            // a transposing read: 16 lanes give the addresses of 4 rows k of 16 columns and get 4 steps of k of a column each
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            const char* p = buf + off + ks * 16 * (ROWS * 2);
            const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
            const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * ROWS * 2)));
            return make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
            const char* p = buf + off + ks * 8 * (ROWS * 4);
            uint4 v;
            v.x = *reinterpret_cast<const unsigned*>(p);
            v.y = *reinterpret_cast<const unsigned*>(p + ROWS * 4);
            v.z = *reinterpret_cast<const unsigned*>(p + 2 * ROWS * 4);
            v.w = *reinterpret_cast<const unsigned*>(p + 3 * ROWS * 4);
            return v;
        }
    }
};

// WM x WN waves; a wave owns MI x 2 accumulators of 32 x 32: rows 32 MI wm .., columns 32 wn .. and BN / 2 + 32 wn .. (GATED: the same
// hidden units of both projections).  A k-tile is 64 bytes deep (32 or 16 steps).  It moves from global memory to LDS without passing
// through registers, into four buffers in turn: the loads of three tiles are in flight while one is multiplied, one barrier a tile.
// With two buffers of twice the depth the product waited for its loads most of the time (0.89 PFLOP/s at 4096 x 2048 x 16384).
// Pieces of 16 bytes are stored at places exclusive-ored with the row, so that the rows that a read serves at once touch all banks.
template <typename T, int WM, int WN, int MI, bool GATED, bool KA, bool KB>
__global__ __launch_bounds__(WM * WN * 64) void gemm_kernel(NtArgs g) {
    constexpr int BM = WM * MI * 32, BN = WN * 64, WAVES = WM * WN, E = 16 / sizeof(T), BK = 64 / sizeof(T);
    constexpr int LOADS = (BM + BN) * 64 / 1024 / WAVES, AUNITS = BM / 16;
    static_assert((BM + BN) * 64 % (1024 * WAVES) == 0 && AUNITS % WAVES == 0 && (!GATED || (KA && KB)), "whole loads");
    static_assert(KA || BM >= 128, "the exclusive or of pieces of rows k needs sixteen of them");
    // separate objects, not one array: the compiler then knows that reads of one do not wait for loads into the others
    __shared__ __attribute__((aligned(1024))) char lds0[(BM + BN) * 64], lds1[(BM + BN) * 64], lds2[(BM + BN) * 64], lds3[(BM + BN) * 64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    // consecutive workgroups go to the 8 dies in turn: give each die a contiguous part of the tiles, walked 4 rows of tiles deep
    int id = blockIdx.x;
    const int tiles = g.mt * g.nt, total = tiles * g.splits;
    {
        const int xcd = id & 7, k = id >> 3, q = total >> 3, r = total & 7;
        id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + k;
    }
    const int split = id / tiles;
    id %= tiles;
    const int deep = 4, band = id / (deep * g.nt), high = min(deep, g.mt - band * deep);
    const int m0 = (band * deep + (id % (deep * g.nt)) % high) * BM, nt = (id % (deep * g.nt)) / high;
    const int n0 = nt * (GATED ? BN / 2 : BN);
    const int kt0 = (int)((long long)g.ktiles * split / g.splits), kt1 = (int)((long long)g.ktiles * (split + 1) / g.splits);

    // load i of a wave fills 1 KB: 16 rows of 64 bytes (k contiguous), or rows k of BM or BN elements
    const char* src[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int unit = i * WAVES + wave;
        if (i * WAVES < AUNITS) {
            if constexpr (KA) {
                const int row = unit * 16 + (lane >> 2), piece = (lane & 3) ^ (lane >> 4);
                src[i] = (const char*)g.A + (long long)min(m0 + row, g.M - 1) * g.a_ld * sizeof(T) + piece * 16;
            } else {
                constexpr int RB = BM * sizeof(T);
                const int k = (unit * 1024 + lane * 16) / RB, piece = (lane * 16 % RB) / 16 ^ (sizeof(T) == 2 ? (k & 3) << 2 : 0);
                src[i] = (const char*)g.A + min(m0 + piece * E, (g.M - 1) / E * E) * sizeof(T);
            }
        } else {
            const int ub = unit - AUNITS;
            if constexpr (KB) {
                const int r = ub * 16 + (lane >> 2), piece = (lane & 3) ^ (lane >> 4);
                const char* p;                                    // rows past the end repeat the last one; their results are not stored
                if (GATED) p = (const char*)(r < BN / 2 ? g.B : g.B1) + (long long)min(n0 + r % (BN / 2), g.N - 1) * g.b_ld * sizeof(T);
                else p = (const char*)g.B + (long long)min(n0 + r, g.N - 1) * g.b_ld * sizeof(T);
                src[i] = p + piece * 16;
            } else {
                constexpr int RB = BN * sizeof(T);
                const int k = (ub * 1024 + lane * 16) / RB, piece = (lane * 16 % RB) / 16 ^ (sizeof(T) == 2 ? (k & 3) << 2 : 0);
                src[i] = (const char*)(unsigned long long)(min(n0 + piece * E, (g.N - 1) / E * E) * sizeof(T));
            }
        }
    }
    auto issue = [&](char* buf, int kt) {
        kt = min(kt, kt1 - 1);         // past the end the last tile again, so that the number of loads in flight stays the same
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int unit = i * WAVES + wave;
            const char* p;
            if (i * WAVES < AUNITS) {
                if constexpr (KA) p = src[i] + (long long)kt * 64;
                else p = src[i] + (long long)min(kt * BK + (unit * 1024 + lane * 16) / (int)(BM * sizeof(T)), g.a_kmax - 1) * g.a_ld * sizeof(T);
            } else {
                if constexpr (KB) p = src[i] + (long long)kt * 64;
                else {
                    const bool second = kt * BK >= g.kcut;
                    const int k = kt * BK - (second ? g.kcut : 0) + ((unit - AUNITS) * 1024 + lane * 16) / (int)(BN * sizeof(T));
                    p = (const char*)(second ? g.B1 : g.B) + (unsigned long long)src[i] + (long long)min(k, g.b_kmax - 1) * g.b_ld * sizeof(T);
                }
            }
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)p,
                                             (__attribute__((address_space(3))) void*)(buf + unit * 1024), 16, 0, 0);
        }
    };
    f32x16 acc[MI][2] = {};
    auto multiply = [&](const char* buf) {
        const Fragment<T, BN, KB> fb0(wn * 32, lane), fb1(BN / 2 + wn * 32, lane);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            const uint4 b0 = fb0.read(buf + BM * 64, ks, lane), b1 = fb1.read(buf + BM * 64, ks, lane);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const Fragment<T, BM, KA> fa((wm * MI + i) * 32, lane);
                const uint4 av = fa.read(buf, ks, lane);
                acc[i][0] = Mma<T>::step(av, b0, acc[i][0]);
                acc[i][1] = Mma<T>::step(av, b1, acc[i][1]);
            }
        }
    };
    // before a tile is read: its loads have arrived (two tiles' may still be in flight), everyone's have, and everyone has read the
    // tile whose buffer is filled next
    auto arrive = [] {
        static_assert(2 * LOADS < 16, "loads that may be in flight: two tiles");
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070 | 2 * LOADS); // vmcnt: two tiles' loads, lgkmcnt 0; as a builtin, so that the compiler counts with it
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if (kt0 < kt1) {
        issue(lds0, kt0);
        issue(lds1, kt0 + 1);
        issue(lds2, kt0 + 2);
    }
    int kt = kt0;
    for (; kt + 4 <= kt1; kt += 4) {
        arrive();
        issue(lds3, kt + 3);
        multiply(lds0);
        arrive();
        issue(lds0, kt + 4);
        multiply(lds1);
        arrive();
        issue(lds1, kt + 5);
        multiply(lds2);
        arrive();
        issue(lds2, kt + 6);
        multiply(lds3);
    }
    if (kt < kt1) {
        arrive();
        issue(lds3, kt + 3);           // (not read: keeps the count)
        multiply(lds0);
        if (kt + 1 < kt1) {
            arrive();
            issue(lds0, kt + 4);
            multiply(lds1);
            if (kt + 2 < kt1) {
                arrive();
                multiply(lds2);
            }
        }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);                // nothing in flight
    __syncthreads();
    // Results: 32 rows at a time through 8 KB of LDS of the wave's own, so that a lane has 8 neighbouring columns; 4-column pieces sit
    // at piece ^ (row & 15) against bank conflicts.
    constexpr int PER = (BM + BN) * 64 / 8192;
    static_assert(4 * PER >= WAVES, "room for the results");
    float* stage = reinterpret_cast<float*>(wave < PER ? lds0 : 2 * PER >= WAVES || wave < 2 * PER ? lds1 : wave < 3 * PER ? lds2 : lds3) + (wave % PER) * 2048;
    const bool wide = g.wide;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int r = 8 * (j >> 2) + 4 * (lane >> 5) + (j & 3), col = c * 32 + (lane & 31);
                stage[r * 64 + (((col >> 2) ^ (r & 15)) << 2) + (col & 3)] = acc[i][c][j];
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int pass = 0; pass < 2; ++pass) {
            const int r = pass * 16 + (lane >> 2), q = lane & 3, m = m0 + (wm * MI + i) * 32 + r;
            float v[2][8];
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float4 t = *reinterpret_cast<const float4*>(&stage[r * 64 + (((c * 8 + q * 2 + h) ^ (r & 15)) << 2)]);
                    v[c][4 * h] = t.x; v[c][4 * h + 1] = t.y; v[c][4 * h + 2] = t.z; v[c][4 * h + 3] = t.w;
                }
            if (m >= g.M) continue;
            if constexpr (GATED) {
                const int n = n0 + wn * 32 + q * 8;
                const long long o = (long long)m * g.N + n;
                float h[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) h[e] = activation(g.act, v[0][e]).x * v[1][e];
                store8((T*)g.out + o, h, g.N - n, wide);
                if (g.pre) {
                    store8(g.pre + o, v[0], g.N - n, wide);
                    store8(g.pre + (long long)g.M * g.N + o, v[1], g.N - n, wide);
                }
            } else {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int n = n0 + c * (BN / 2) + wn * 32 + q * 8;
                    if (g.part) store8(g.part + ((long long)split * g.M + m) * g.N + n, v[c], g.N - n, wide);
                    else if (m < g.cut ? m < g.rows : m - g.cut < g.rows)
                        store8((T*)(m < g.cut ? g.out : g.out1) + (long long)(m < g.cut ? m : m - g.cut) * g.N + n, v[c], g.N - n, wide);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// out = sum of the splits' partial products, in order
template <typename T>
__global__ __launch_bounds__(256) void gemm_join_kernel(NtArgs g) {
    const long long total = (long long)g.M * g.N;
    for (long long o = (long long)blockIdx.x * 256 + threadIdx.x; o < total; o += 256ll * gridDim.x) {
        float v = 0.f;
        for (int k = 0; k < g.splits; ++k) v += g.part[k * total + o];
        const int m = (int)(o / g.N), r = m < g.cut ? m : m - g.cut;
        if (r < g.rows) ((T*)(m < g.cut ? g.out : g.out1))[(long long)r * g.N + o % g.N] = (T)v;
    }
}

// ---- few rows --------------------------------------------------------------------------------------------------------
// Few rows of x, or few products altogether.  A workgroup owns 16 hidden units of both projections and 16 MB rows (blockIdx.y) and
// shares the contraction among its waves, whose partial products are joined through LDS in wave order.  Up to 64 rows the weights are
// read once, which is the time; operands go from memory to the matrix cores without LDS, any alignment.
struct FewArgs {
    const void *x, *wg, *wu;
    long long x_ld, w_ld;
    int M, K, F, act;
    void* h;
    float* pre;
};

template <typename T>
struct Mma16;
template <>
struct Mma16<bf16> {
    static __device__ __forceinline__ f32x4 step(uint4 a, uint4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma16<f16> {
    static __device__ __forceinline__ f32x4 step(uint4 a, uint4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma16<float> {
    static __device__ __forceinline__ f32x4 step(uint4 a, uint4 b, f32x4 c) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
        return c;
    }
};

// 16 bytes of a row from element k on, zero past its end.  Unaligned rows are read as the dwords that hold the piece (each holds a valid
// element, so that none lies outside the matrix's memory) and shifted; only a row's last piece goes element by element.
typedef unsigned u32x4_dword __attribute__((ext_vector_type(4), aligned(4)));
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 row_piece(const T* row, int k, int K, bool ok) {
    constexpr int E = 16 / sizeof(T);
    uint4 v = make_uint4(0, 0, 0, 0);
    if constexpr (ALIGNED) {           // whole pieces: K is a multiple of E
        if (ok && k < K) v = *reinterpret_cast<const uint4*>(row + k);
    } else if (ok && k + E <= K) {
        const unsigned long long a = (unsigned long long)(row + k);
        const unsigned* p = (const unsigned*)(a & ~3ull);
        const u32x4_dword d = *(const u32x4_dword*)p;
        if constexpr (sizeof(T) == 4) {
            v = make_uint4(d.x, d.y, d.z, d.w);
        } else {
            const unsigned shift = (unsigned)(a & 2) * 8, last = p[shift ? 4 : 3];
            v.x = __builtin_amdgcn_alignbit(d.y, d.x, shift);
            v.y = __builtin_amdgcn_alignbit(d.z, d.y, shift);
            v.z = __builtin_amdgcn_alignbit(d.w, d.z, shift);
            v.w = __builtin_amdgcn_alignbit(last, d.w, shift);
        }
    } else if (ok && k < K) {
        Vec<T, E> t;
#pragma unroll
        for (int i = 0; i < E; ++i) t.v[i] = k + i < K ? row[k + i] : (T)0.f;
        v = __builtin_bit_cast(uint4, t);
    }
    return v;
}

template <typename T, int MB, bool ALIGNED>
__global__ __launch_bounds__(1024) void gated_few_kernel(FewArgs g) {
    constexpr int E = 16 / sizeof(T), BK = 4 * E, UN = MB == 1 ? 4 : 2;
    extern __shared__ f32x4 red[];     // [waves][2 MB][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, f = blockIdx.x * 16 + r, m0 = blockIdx.y * 16 * MB;
    const bool okf = f < g.F;
    const T* wg = (const T*)g.wg + (long long)(okf ? f : 0) * g.w_ld;
    const T* wu = (const T*)g.wu + (long long)(okf ? f : 0) * g.w_ld;
    const int steps = (g.K + BK - 1) / BK, s0 = steps * wave / waves, s1 = steps * (wave + 1) / waves;
    f32x4 acc[2][MB] = {};
    const T* xr[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) xr[b] = (const T*)g.x + (long long)min(m0 + b * 16 + r, g.M - 1) * g.x_ld;
    for (int s = s0; s < s1; s += UN) {
        uint4 a0[UN], a1[UN], bx[UN][MB];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int k = s + i < s1 ? (s + i) * BK + (lane >> 4) * E : g.K;
            a0[i] = row_piece<T, ALIGNED>(wg, k, g.K, okf);
            a1[i] = row_piece<T, ALIGNED>(wu, k, g.K, okf);
#pragma unroll
            for (int b = 0; b < MB; ++b) bx[i][b] = row_piece<T, ALIGNED>(xr[b], k, g.K, m0 + b * 16 + r < g.M);
        }
#pragma unroll
        for (int i = 0; i < UN; ++i)
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                acc[0][b] = Mma16<T>::step(a0[i], bx[i][b], acc[0][b]);
                acc[1][b] = Mma16<T>::step(a1[i], bx[i][b], acc[1][b]);
            }
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        red[(wave * 2 * MB + b) * 64 + lane] = acc[0][b];
        red[(wave * 2 * MB + MB + b) * 64 + lane] = acc[1][b];
    }
    __syncthreads();
    for (int e = threadIdx.x; e < MB * 64; e += blockDim.x) {
        f32x4 gate = {}, up = {};
        for (int w = 0; w < waves; ++w) {
            gate += red[w * 2 * MB * 64 + e];
            up += red[(w * 2 * MB + MB) * 64 + e];
        }
        const int m = m0 + (e >> 6) * 16 + (e & 15);
        if (m >= g.M) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int n = blockIdx.x * 16 + 4 * ((e & 63) >> 4) + j;
            if (n >= g.F) continue;
            const long long o = (long long)m * g.F + n;
            ((T*)g.h)[o] = (T)(activation(g.act, gate[j]).x * up[j]);
            if (g.pre) { g.pre[o] = gate[j]; g.pre[(long long)g.M * g.F + o] = up[j]; }
        }
    }
}

// ---- operands laid out for the products ------------------------------------------------------------------------------
// up to three matrices: dst[row][0 .. ld): src row, zero from `cols` on
struct PadArgs {
    const void* src[3];
    long long s_ld[3];
    void* dst[3];
    int rows[3], cols, ld;
};
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(PadArgs p) {
    constexpr int E = 16 / sizeof(T);
    const int k = blockIdx.y;
    const unsigned pieces = (unsigned)(p.ld / E);
    const long long total = (long long)p.rows[k] * pieces;
    for (long long o = (long long)blockIdx.x * 256 + threadIdx.x; o < total; o += 256ll * gridDim.x) {
        const long long row = total < (1ll << 32) ? (unsigned)o / pieces : o / pieces;
        const int c = (int)(o - row * pieces) * E;
        *reinterpret_cast<uint4*>((T*)p.dst[k] + row * p.ld + c) = row_piece<T, false>((const T*)p.src[k] + row * p.s_ld[k], c, p.cols, true);
    }
}

// zeros
template <typename T>
__global__ __launch_bounds__(256) void zero_kernel(T* p, long long n) {
    for (long long o = (long long)blockIdx.x * 256 + threadIdx.x; o < n; o += 256ll * gridDim.x) p[o] = (T)0.f;
}

// dG, dU from the saved projections: rows [Mp][2 Fp], dG then dU, zero past M and past F.  Bound by memory (2 e + 2 e + 8 + e bytes an
// element): eight elements a thread; VEC: rows of pre and dh may be read in pieces of 16 bytes.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void gate_slope_kernel(int M, int F, int Mp, int Fp, int act, const float* pre, const T* dh, long long dh_ld, T* rows) {
    constexpr int E = 16 / sizeof(T);
    const unsigned cols = Fp / 8, m = blockIdx.x / ((cols + 255) / 256), c = blockIdx.x % ((cols + 255) / 256) * 256 + threadIdx.x;
    if (c >= cols) return;
    const int f = c * 8;
    const long long o = (long long)m * F + f, total = (long long)M * F;
    float g[8], u[8];
    T d[8], vg[8], vu[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) { g[i] = u[i] = 0.f; d[i] = (T)0.f; }
    if ((int)m < M) {
        if constexpr (VEC) {
            if (f < F) {               // F is a multiple of 8
                *(float4*)g = *(const float4*)(pre + o); *(float4*)(g + 4) = *(const float4*)(pre + o + 4);
                *(float4*)u = *(const float4*)(pre + total + o); *(float4*)(u + 4) = *(const float4*)(pre + total + o + 4);
#pragma unroll
                for (int i = 0; i < 8; i += E) *(Vec<T, E>*)(d + i) = load_vec<T, E>(dh + (long long)m * dh_ld + f + i);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (f + i < F) { g[i] = pre[o + i]; u[i] = pre[total + o + i]; d[i] = dh[(long long)m * dh_ld + f + i]; }
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 a = activation(act, g[i]);
        const bool in = (int)m < M && f + i < F;
        vg[i] = (T)(in ? (float)d[i] * u[i] * a.y : 0.f);
        vu[i] = (T)(in ? (float)d[i] * a.x : 0.f);
    }
    T* out = rows + (long long)m * 2 * Fp + f;
#pragma unroll
    for (int i = 0; i < 8; i += E) {
        store_vec(out + i, *(const Vec<T, E>*)(vg + i));
        store_vec(out + Fp + i, *(const Vec<T, E>*)(vu + i));
    }
}

static int ffn_check(const char* what, int dtype, int M, int K, int F, int act) {
    NMPC_REQUIRE(dtype >= NMPC_F32 && dtype <= NMPC_F16, "%s: unknown element type %d", what, dtype);
    NMPC_REQUIRE(M >= 0 && K >= 1 && F >= 1, "%s: bad sizes (%d rows, %d inputs, %d hidden units)", what, M, K, F);
    NMPC_REQUIRE(act >= NMPC_ACT_SILU && act <= NMPC_ACT_SIGMOID, "%s: activation %d", what, act);
    NMPC_REQUIRE(M < (1 << 22) && K < (1 << 21) && F < (1 << 21), "%s: at most 2^22 rows and 2^21 inputs and hidden units", what);
    // a launch has fewer than 2^32 threads
    NMPC_REQUIRE((M + 64ll) * (F / 2048 + 1) < (1 << 24), "%s: too many elements for one launch", what);
    return 0;
}
static unsigned long long round256(unsigned long long v) { return (v + 255) / 256 * 256; }

constexpr int FEW_ROWS = 64;

template <typename T>
constexpr int ktile() { return 64 / (int)sizeof(T); }
static int up_to(int v, int m) { return (v + m - 1) / m * m; }

// whether a matrix with rows of K elements can be read in pieces of 16 bytes as it is; by k: in whole k-tiles
template <typename T>
static bool tiled(const void* p, long long ld, int K, bool by_k) {
    return K % (by_k ? ktile<T>() : 16 / (int)sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * sizeof(T) % 16 == 0;
}

// Tile size and splits of a product: the choice of least estimated time.  A 256 x 256 tile has a CU for itself, two 128 x 128 tiles share
// one; a k-tile of the large one takes 1.06 us in 16 bits and 4.0 us in fp32 (measured at 16384 x 2048 x 4096), of the small one a
// quarter of it and a sixth more, less well used where a CU has one alone.  Tiles of 64 x 128 (`small`: A's rows lie along k) divide few
// rows more finely and cost 0.24 and 0.60 us a k-tile: 512 x 2048 x 2048 in bf16 19 instead of 24 us, 256 x 1024 x 4096 in fp32 42 instead
// of 71; at 1024 x 1024 x 4096 they take 37 instead of 29 and 142 instead of 139.  Every round of tiles pays for filling and draining;
// a split contraction pays for writing and reading its partial products.
struct Shape {
    int bm, bn, splits;
    double us;
};
template <typename T>
static Shape product_shape(int M, int N, int ktiles, bool small, bool may_split) {
    const double ktime = sizeof(T) == 2 ? 1.06 : 4.0, fill = 4.0;
    Shape best = {128, 128, 1, 1e30};
    for (int tile = small ? 0 : 1; tile < 3; ++tile) {
        const int bm = tile == 0 ? 64 : tile == 1 ? 128 : 256, bn = tile == 2 ? 256 : 128;
        const double tiles = (double)((M + bm - 1) / bm) * ((N + bn - 1) / bn);
        for (int splits = 1; splits <= (may_split ? 64 : 1) && (splits == 1 || splits * 4 <= ktiles); ++splits) {
            const double n = tiles * splits, depth = (ktiles + splits - 1) / splits;
            double t;
            if (tile == 2) t = ceil(n / 256) * (depth * ktime + fill);
            else if (tile == 1) t = n <= 256 ? depth * ktime * 0.25 * (sizeof(T) == 2 ? 1.25 : 1.0) + fill : ceil(n / 512) * (depth * ktime * 0.5 * 1.17 + fill);
            else t = ceil(n / 256) * depth * (sizeof(T) == 2 ? 0.24 : 0.60) + fill;
            if (splits > 1) t += 6.0 + (double)splits * M * N * 8 / 4.5e6;
            if (t < best.us) best = {bm, bn, splits, t};
        }
    }
    return best;
}

// How the kernel for few rows would run a forward pass: rows of a workgroup as many as leave every CU one (at most 64: the weights are
// read once for them), and its estimated time.  A step of 64 bytes of k of 64 rows x 16 units takes 0.68 ns of the chip in 16 bits (the
// rate of the cache lines its loads touch) and 1.03 ns in fp32 (its products), 1.0 and 1.2 ns on unaligned rows; measured at
// 512 x 2048 x 2048 and 333 x 1001 x 2731.
struct FewShape {
    int mb, waves;
    dim3 grid;
    double us;
};
template <typename T>
static FewShape few_shape(int M, int K, int F, bool aligned) {
    FewShape s = {4, 4, dim3((F + 15) / 16, 1), 0.0};
    auto rows = [&] { return (M + 16 * s.mb - 1) / (16 * s.mb); };
    while (s.mb > 1 && (8 * s.mb >= M || (long long)s.grid.x * rows() < 256)) s.mb /= 2;
    s.grid.y = rows();
    const double blocks = (double)s.grid.x * s.grid.y;
    while (s.waves < (s.mb == 4 ? 8 : 16) && blocks * s.waves < 2048) s.waves *= 2;
    const double ns = sizeof(T) == 2 ? (aligned ? 0.68 : 1.0) : (aligned ? 1.03 : 1.2);
    const double steps = blocks * ((K + ktile<T>() - 1) / ktile<T>()) * (sizeof(T) == 2 ? (2 + s.mb) / 6.0 : s.mb / 4.0);
    s.us = 4.0 + steps * ns * 1e-3 * (blocks < 256 ? 256 / blocks : 1.0);
    return s;
}

// Does it?  Up to 64 rows always; beyond, where its estimate is below that of the tiles, which leave most CUs idle when there are few of
// them and need copies of unaligned operands.
template <typename T>
static bool serves_few(int M, int K, int F, bool aligned) {
    if (M <= FEW_ROWS) return true;
    if ((M + 15) / 16 > 65535) return false;
    return few_shape<T>(M, K, F, aligned).us < product_shape<T>(M, 2 * F, (K + ktile<T>() - 1) / ktile<T>(), true, false).us + (aligned ? 0.0 : 6.0);
}

template <typename T, bool GATED, bool KA, bool KB>
static int run_product(NtArgs g, hipStream_t st) {
    const int cols = GATED ? 2 * g.N : g.N;
    const Shape shape = product_shape<T>(g.M, cols, g.ktiles, KA, !GATED && g.part);
    g.splits = shape.splits;
    if (g.splits == 1) g.part = nullptr;
    g.wide = g.N % 8 == 0 && ((uintptr_t)g.out | (uintptr_t)g.out1 | (uintptr_t)g.pre) % 16 == 0;
    const int bn = GATED ? shape.bn / 2 : shape.bn;
    g.mt = (g.M + shape.bm - 1) / shape.bm;
    g.nt = (g.N + bn - 1) / bn;
    const long long grid = (long long)g.mt * g.nt * g.splits;
    NMPC_REQUIRE(grid < (1 << 22), "gated_ffn: too many tiles for one launch");
    if (shape.bm == 256) gemm_kernel<T, 2, 4, 4, GATED, KA, KB><<<(unsigned)grid, 512, 0, st>>>(g);
    else if (shape.bm == 64) {
        if constexpr (KA) gemm_kernel<T, 2, 2, 1, GATED, KA, KB><<<(unsigned)grid, 256, 0, st>>>(g);
    } else gemm_kernel<T, 2, 2, 2, GATED, KA, KB><<<(unsigned)grid, 256, 0, st>>>(g);
    if (g.splits > 1) {
        const long long blocks = ((long long)g.M * g.N + 255) / 256;
        gemm_join_kernel<T><<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, st>>>(g);
    }
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}

static unsigned pad_grid(long long total) {
    const long long blocks = (total + 255) / 256;
    return (unsigned)(blocks < 8192 ? blocks : 8192);
}

// Which kernel a product takes: the forward pass (0), dx (1) or [dWg; dWu] (2).
template <typename T>
static Shape shape_of(int M, int K, int F, int product, bool copy) {
    const int kt = ktile<T>(), Fp = up_to(F, kt), Mp = up_to(M, kt);
    if (product == 1) return product_shape<T>(M, K, 2 * Fp / kt, true, true);
    if (product == 2) return product_shape<T>(2 * Fp, K, Mp / kt, false, true);
    const bool aligned = !copy && K % kt == 0;
    if (!serves_few<T>(M, K, F, aligned)) return product_shape<T>(M, 2 * F, (K + kt - 1) / kt, true, false);
    const FewShape fs = few_shape<T>(M, K, F, !copy && K % (16 / (int)sizeof(T)) == 0);
    return {16 * fs.mb, 32, fs.waves, fs.us};
}

// The workspace of a call: copies of operands that cannot be read in pieces as they are, and the gradient's intermediates.
struct FfnSpace {
    unsigned long long bytes, x, wg, wu, rows, part;
    int Kp;                            // row length of the copies
    template <typename T>
    static FfnSpace plan(int M, int K, int F, bool backward, bool copy) {
        FfnSpace s = {};
        const unsigned long long e = sizeof(T);
        const int kt = ktile<T>(), Fp = up_to(F, kt), Mp = up_to(M, kt);
        auto take = [&](unsigned long long bytes) { const unsigned long long at = s.bytes; s.bytes += round256(bytes); return at; };
        s.Kp = up_to(K, backward ? 16 / (int)e : kt);
        if ((copy || K != s.Kp) && (backward || !serves_few<T>(M, K, F, false))) {
            s.x = take(e * M * s.Kp);
            s.wg = take(e * F * s.Kp);
            s.wu = take(e * F * s.Kp);
        }
        if (!backward) return s;
        s.rows = take(e * Mp * 2 * Fp);
        const Shape a = shape_of<T>(M, K, F, 1, copy), b = shape_of<T>(M, K, F, 2, copy);
        const unsigned long long pa = a.splits > 1 ? 4ull * a.splits * M * K : 0, pb = b.splits > 1 ? 4ull * b.splits * 2 * Fp * K : 0;
        s.part = take(pa > pb ? pa : pb);
        return s;
    }
};

// the operands of a product as they are, or their copies in the workspace
template <typename T>
static int lay_out(const FfnSpace& sp, bool by_k, int M, int K, int F, const void*& x, long long& x_ld, const void*& wg, const void*& wu, long long& w_ld,
                   char* ws, hipStream_t st) {
    if (tiled<T>(x, x_ld, K, by_k) && tiled<T>(wg, w_ld, K, by_k) && tiled<T>(wu, w_ld, K, by_k)) return 0;
    const int Kp = sp.Kp;
    const PadArgs p = {{x, wg, wu}, {x_ld, w_ld, w_ld}, {ws + sp.x, ws + sp.wg, ws + sp.wu}, {M, F, F}, K, Kp};
    pad_kernel<T><<<dim3(pad_grid((long long)(M > F ? M : F) * Kp * (long long)sizeof(T) / 16), 3), 256, 0, st>>>(p);
    NMPC_HIP_CHECK(hipGetLastError());
    x = ws + sp.x; wg = ws + sp.wg; wu = ws + sp.wu;
    x_ld = w_ld = Kp;
    return 0;
}

template <typename T>
static int run_forward(int M, int K, int F, const void* x, long long x_ld, const void* wg, const void* wu, long long w_ld, int act, void* h,
                       float* pre, char* ws, unsigned long long ws_bytes, hipStream_t st) {
    const bool copy = !(tiled<T>(x, x_ld, K, true) && tiled<T>(wg, w_ld, K, true) && tiled<T>(wu, w_ld, K, true));
    const FfnSpace sp = FfnSpace::plan<T>(M, K, F, false, copy);
    NMPC_REQUIRE(sp.bytes == 0 || (ws && ws_bytes >= sp.bytes), "nmpc_gated_ffn: workspace of %llu bytes, %llu needed", ws_bytes, sp.bytes);
    if (serves_few<T>(M, K, F, !copy)) {
        constexpr int E = 16 / sizeof(T);
        FewArgs g = {x, wg, wu, x_ld, w_ld, M, K, F, act, h, pre};
        const bool al = K % E == 0 && vec_ok<T>(x, x_ld, 0, E) && vec_ok<T>(wg, w_ld, 0, E) && vec_ok<T>(wu, w_ld, 0, E);
        const FewShape fs = few_shape<T>(M, K, F, al);
        const dim3 grid = fs.grid;
        const int mb = fs.mb, waves = fs.waves;
        const unsigned shared = waves * 2 * mb * 64 * 16;
#define NMPC_FEW(MB_)                                                                                                   \
    if (al) gated_few_kernel<T, MB_, true><<<grid, waves * 64, shared, st>>>(g);                                        \
    else gated_few_kernel<T, MB_, false><<<grid, waves * 64, shared, st>>>(g);
        if (mb == 1) { NMPC_FEW(1) } else if (mb == 2) { NMPC_FEW(2) } else { NMPC_FEW(4) }
#undef NMPC_FEW
        NMPC_HIP_CHECK(hipGetLastError());
        return 0;
    }
    if (lay_out<T>(sp, true, M, K, F, x, x_ld, wg, wu, w_ld, ws, st)) return 1;
    NtArgs g = {};
    g.M = M; g.N = F; g.act = act; g.out = h; g.pre = pre;
    g.ktiles = sp.Kp / ktile<T>();
    g.A = x; g.a_ld = x_ld; g.B = wg; g.B1 = wu; g.b_ld = w_ld;
    return run_product<T, true, true, true>(g, st);
}

template <typename T>
static int run_backward(int M, int K, int F, const void* x, long long x_ld, const void* wg, const void* wu, long long w_ld, int act,
                        const float* pre, const void* dh, long long dh_ld, void* dx, void* dwg, void* dwu, char* ws,
                        unsigned long long ws_bytes, hipStream_t st) {
    if (M == 0) {
        zero_kernel<T><<<pad_grid((long long)F * K), 256, 0, st>>>((T*)dwg, (long long)F * K);
        zero_kernel<T><<<pad_grid((long long)F * K), 256, 0, st>>>((T*)dwu, (long long)F * K);
        NMPC_HIP_CHECK(hipGetLastError());
        return 0;
    }
    const bool copy = !(tiled<T>(x, x_ld, K, false) && tiled<T>(wg, w_ld, K, false) && tiled<T>(wu, w_ld, K, false));
    const FfnSpace sp = FfnSpace::plan<T>(M, K, F, true, copy);
    NMPC_REQUIRE(ws && ws_bytes >= sp.bytes, "nmpc_gated_ffn_bwd: workspace of %llu bytes, %llu needed", ws_bytes, sp.bytes);
    if (lay_out<T>(sp, false, M, K, F, x, x_ld, wg, wu, w_ld, ws, st)) return 1;
    const int kt = ktile<T>(), Fp = up_to(F, kt), Mp = up_to(M, kt);
    T* rows = (T*)(ws + sp.rows);
    constexpr int E = 16 / sizeof(T);
    const unsigned grid = (unsigned)Mp * (unsigned)((Fp / 8 + 255) / 256);
    if (F % 8 == 0 && vec_ok<float>(pre, 0, 0, 4) && vec_ok<T>(dh, dh_ld, 0, E))
        gate_slope_kernel<T, true><<<grid, 256, 0, st>>>(M, F, Mp, Fp, act, pre, (const T*)dh, dh_ld, rows);
    else gate_slope_kernel<T, false><<<grid, 256, 0, st>>>(M, F, Mp, Fp, act, pre, (const T*)dh, dh_ld, rows);
    NtArgs g = {};                     // dx = [dG dU] [Wg; Wu]
    g.A = rows; g.a_ld = 2 * Fp; g.B = wg; g.B1 = wu; g.b_ld = w_ld;
    g.M = M; g.N = K; g.ktiles = 2 * Fp / kt; g.kcut = Fp; g.b_kmax = F;
    g.out = dx; g.cut = g.rows = M; g.part = (float*)(ws + sp.part);
    if (run_product<T, false, true, false>(g, st)) return 1;
    g = NtArgs{};                      // [dWg; dWu] = [dG dU]' x
    g.A = rows; g.a_ld = 2 * Fp; g.a_kmax = Mp; g.B = x; g.b_ld = x_ld; g.kcut = Mp; g.b_kmax = M;
    g.M = 2 * Fp; g.N = K; g.ktiles = Mp / kt;
    g.out = dwg; g.out1 = dwu; g.cut = Fp; g.rows = F; g.part = (float*)(ws + sp.part);
    return run_product<T, false, false, false>(g, st);
}

}  // namespace nmpc

using namespace nmpc;

extern "C" unsigned long long nmpc_gated_ffn_workspace_bytes(int dtype, int M, int K, int F, int backward, int copy) {
    if (M <= 0 || K <= 0 || F <= 0) return 0;
    return dtype == NMPC_F32 ? FfnSpace::plan<float>(M, K, F, backward != 0, copy != 0).bytes
                             : FfnSpace::plan<bf16>(M, K, F, backward != 0, copy != 0).bytes;
}

extern "C" int nmpc_gated_ffn_plan(int dtype, int M, int K, int F, int product, int copy, int shape[3]) {
    if (ffn_check("nmpc_gated_ffn_plan", dtype, M, K, F, NMPC_ACT_SILU)) return 1;
    NMPC_REQUIRE(M >= 1 && product >= 0 && product <= 2 && shape, "nmpc_gated_ffn_plan: bad argument");
    const Shape s = dtype == NMPC_F32 ? shape_of<float>(M, K, F, product, copy != 0) : shape_of<bf16>(M, K, F, product, copy != 0);
    shape[0] = s.bm; shape[1] = s.bn; shape[2] = s.splits;
    return 0;
}

extern "C" int nmpc_gated_ffn(int dtype, int M, int K, int F, const void* x, long long x_ld, const void* wg, long long wg_ld,
                              const void* wu, long long wu_ld, int act, void* h, float* pre, void* workspace,
                              unsigned long long workspace_bytes, void* stream) {
    if (ffn_check("nmpc_gated_ffn", dtype, M, K, F, act)) return 1;
    if (M == 0) return 0;
    NMPC_REQUIRE(x && wg && wu && h, "nmpc_gated_ffn: null argument");
    NMPC_REQUIRE(wg_ld == wu_ld, "nmpc_gated_ffn: the weight matrices have different row strides");
    NMPC_REQUIRE((uintptr_t)workspace % 16 == 0, "nmpc_gated_ffn: the workspace starts on 16 bytes");
    NMPC_DTYPE_SWITCH(dtype, { return run_forward<T_>(M, K, F, x, x_ld, wg, wu, wg_ld, act, h, pre, (char*)workspace, workspace_bytes, (hipStream_t)stream); })
    return 0;
}

extern "C" int nmpc_gated_ffn_bwd(int dtype, int M, int K, int F, const void* x, long long x_ld, const void* wg, long long wg_ld,
                                  const void* wu, long long wu_ld, int act, const float* pre, const void* dh, long long dh_ld, void* dx,
                                  void* dwg, void* dwu, void* workspace, unsigned long long workspace_bytes, void* stream) {
    if (ffn_check("nmpc_gated_ffn_bwd", dtype, M, K, F, act)) return 1;
    NMPC_REQUIRE(dwg && dwu && (M == 0 || (x && wg && wu && pre && dh && dx)), "nmpc_gated_ffn_bwd: null argument");
    NMPC_REQUIRE(wg_ld == wu_ld, "nmpc_gated_ffn_bwd: the weight matrices have different row strides");
    NMPC_REQUIRE((uintptr_t)workspace % 16 == 0, "nmpc_gated_ffn_bwd: the workspace starts on 16 bytes");
    NMPC_DTYPE_SWITCH(dtype, { return run_backward<T_>(M, K, F, x, x_ld, wg, wu, wg_ld, act, pre, dh, dh_ld, dx, dwg, dwu, (char*)workspace, workspace_bytes, (hipStream_t)stream); })
    return 0;
}
