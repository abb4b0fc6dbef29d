// Gated feed-forward projections: h = act(x Wg') o (x Wu'), x[M,K], Wg / Wu[F,K], and their gradients
//   dG = dh o up o act'(gate),  dU = dh o act(gate),
//   dx = dG Wg + dU Wu,  dWg = dG' x,  dWu = dU' x.
// Both projections of a tile are accumulated side by side, so that the activation and the product happen in registers and
// neither projection is written (a training pass keeps both in fp32 for the gradient).  Products run on the matrix cores with
// fp32 accumulation; dG and dU are rounded to the element type once, as operands of the next products.
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
// out[m][n] = sum_k A[m][k] B[n][k], both operands with contiguous rows of whole 128-byte k-tiles.
struct NtArgs {
    const void *A, *B, *B1;            // GATED: B and B1 are the two weight matrices
    long long a_ld, b_ld;              // elements
    int M, N, ktiles, act;
    void *out, *out1;                  // rows from `cut` on go to out1 (two gradients of one product)
    int cut;
    float* pre;                        // GATED: [2][M][N], both projections, may be null
    float* part;                       // fp32 partial products [splits][M][N] instead of out
    int splits;
    int mt, nt;                        // tiles
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

// WM x WN waves; a wave owns MI x 2 accumulators of 32 x 32: rows 32 MI wm .., columns 32 wn .. and BN / 2 + 32 wn .. (GATED: the same
// hidden units of both projections).  A k-tile is a row of 128 bytes, moved from global memory to LDS without passing through
// registers, into two buffers in turn: the loads of the next tile are in flight while this one is multiplied.  Within a row the
// 16-byte pieces sit at piece ^ (row & 7), so that the 8 rows that a read serves at once touch all banks.
template <typename T, int WM, int WN, int MI, bool GATED>
__global__ __launch_bounds__(WM * WN * 64) void gemm_nt_kernel(NtArgs g) {
    constexpr int BM = WM * MI * 32, BN = WN * 64, WAVES = WM * WN, ROWS = BM + BN, LOADS = ROWS / 8 / WAVES;
    static_assert(ROWS % (8 * WAVES) == 0 && BM % 8 == 0, "whole loads");
    // two objects, not one array: the compiler then knows that reads of one do not wait for loads into the other
    __shared__ __attribute__((aligned(1024))) char lds0[ROWS * 128], lds1[ROWS * 128];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
    // consecutive workgroups go to the 8 dies in turn: give each die a contiguous part of the tiles, walked 8 rows of tiles deep
    int id = blockIdx.x;
    const int tiles = g.mt * g.nt, total = tiles * g.splits;
    {
        const int xcd = id & 7, k = id >> 3, q = total >> 3, r = total & 7;
        id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + k;
    }
    const int split = id / tiles;
    id %= tiles;
    const int deep = 8, band = id / (deep * g.nt), high = min(deep, g.mt - band * deep);
    const int m0 = (band * deep + (id % (deep * g.nt)) % high) * BM, nt = (id % (deep * g.nt)) / high;
    const int n0 = nt * (GATED ? BN / 2 : BN);
    const int kt0 = (int)((long long)g.ktiles * split / g.splits), kt1 = (int)((long long)g.ktiles * (split + 1) / g.splits);

    const char* src[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int row = (i * WAVES + wave) * 8 + (lane >> 3), piece = (lane & 7) ^ (lane >> 3);
        const char* p;
        if (row < BM) {
            p = (const char*)g.A + (long long)min(m0 + row, g.M - 1) * g.a_ld * sizeof(T);
        } else {                       // rows past the end repeat the last one; their results are not stored
            const int r = row - BM;
            if (GATED) p = (const char*)(r < BN / 2 ? g.B : g.B1) + (long long)min(n0 + r % (BN / 2), g.N - 1) * g.b_ld * sizeof(T);
            else p = (const char*)g.B + (long long)min(n0 + r, g.N - 1) * g.b_ld * sizeof(T);
        }
        src[i] = p + piece * 16 + (long long)kt0 * 128;
    }
    auto issue = [&](char* buf) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src[i],
                                             (__attribute__((address_space(3))) void*)(buf + (i * WAVES + wave) * 1024), 16, 0, 0);
            src[i] += 128;
        }
    };
    f32x16 acc[MI][2] = {};
    auto multiply = [&](const char* buf) {
        const char* a = buf + (wm * MI * 32 + (lane & 31)) * 128;
        const char* b = buf + (BM + wn * 32 + (lane & 31)) * 128;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
            const int piece = ((ks * 2 + (lane >> 5)) ^ (lane & 7)) * 16;
            const uint4 b0 = *reinterpret_cast<const uint4*>(b + piece), b1 = *reinterpret_cast<const uint4*>(b + BN / 2 * 128 + piece);
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const uint4 av = *reinterpret_cast<const uint4*>(a + i * 32 * 128 + piece);
                acc[i][0] = Mma<T>::step(av, b0, acc[i][0]);
                acc[i][1] = Mma<T>::step(av, b1, acc[i][1]);
            }
        }
    };
    // before a tile is read: its loads (counted as memory loads) have arrived, and everyone is done with the other buffer
    auto arrive = [] {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    if (kt0 < kt1) issue(lds0);
    int kt = kt0;
    for (; kt + 2 <= kt1; kt += 2) {
        arrive();
        issue(lds1);
        multiply(lds0);
        arrive();
        if (kt + 2 < kt1) issue(lds0);
        multiply(lds1);
    }
    if (kt < kt1) {
        arrive();
        multiply(lds0);
    }
    __syncthreads();
    // Results: 32 rows at a time through 8 KB of LDS of the wave's own, so that a lane has 8 neighbouring columns; 4-column pieces sit
    // at piece ^ (row & 15) against bank conflicts.
    float* stage = reinterpret_cast<float*>(lds0) + wave * 2048;
    const bool wide = g.N % 8 == 0;
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
                    else if (m < g.cut) store8((T*)g.out + (long long)m * g.N + n, v[c], g.N - n, wide);
                    else store8((T*)g.out1 + (long long)(m - g.cut) * g.N + n, v[c], g.N - n, wide);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// out = sum of the splits' partial products, in order
template <typename T>
__global__ __launch_bounds__(256) void gemm_join_kernel(NtArgs g) {
    const long long total = (long long)g.M * g.N, cut = (long long)g.cut * g.N;
    for (long long o = (long long)blockIdx.x * 256 + threadIdx.x; o < total; o += 256ll * gridDim.x) {
        float v = 0.f;
        for (int k = 0; k < g.splits; ++k) v += g.part[k * total + o];
        if (o < cut) ((T*)g.out)[o] = (T)v;
        else ((T*)g.out1)[o - cut] = (T)v;
    }
}

// ---- few rows --------------------------------------------------------------------------------------------------------
// Up to 64 rows of x: the weights are read once, which is the time.  A workgroup owns 16 hidden units of both projections and
// shares the contraction among its waves; their partial products are joined through LDS in wave order.
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

// 16 bytes of a row from element k on, zero past its end
template <typename T, bool ALIGNED>
__device__ __forceinline__ uint4 row_piece(const T* row, int k, int K, bool ok) {
    constexpr int E = 16 / sizeof(T);
    if constexpr (ALIGNED) {           // whole pieces: K is a multiple of E
        if (ok && k < K) return *reinterpret_cast<const uint4*>(row + k);
        return make_uint4(0, 0, 0, 0);
    } else {
        Vec<T, E> v;
#pragma unroll
        for (int i = 0; i < E; ++i) v.v[i] = ok && k + i < K ? row[k + i] : (T)0.f;
        return __builtin_bit_cast(uint4, v);
    }
}

template <typename T, int MB, bool ALIGNED>
__global__ __launch_bounds__(1024) void gated_few_kernel(FewArgs g) {
    constexpr int E = 16 / sizeof(T), BK = 4 * E, UN = MB == 1 ? 4 : 2;
    extern __shared__ f32x4 red[];     // [waves][2 MB][64]
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const int r = lane & 15, f = blockIdx.x * 16 + r;
    const bool okf = f < g.F;
    const T* wg = (const T*)g.wg + (long long)(okf ? f : 0) * g.w_ld;
    const T* wu = (const T*)g.wu + (long long)(okf ? f : 0) * g.w_ld;
    const int steps = (g.K + BK - 1) / BK, s0 = steps * wave / waves, s1 = steps * (wave + 1) / waves;
    f32x4 acc[2][MB] = {};
    const T* xr[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) xr[b] = (const T*)g.x + (long long)min(b * 16 + r, g.M - 1) * g.x_ld;
    for (int s = s0; s < s1; s += UN) {
        uint4 a0[UN], a1[UN], bx[UN][MB];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int k = s + i < s1 ? (s + i) * BK + (lane >> 4) * E : g.K;
            a0[i] = row_piece<T, ALIGNED>(wg, k, g.K, okf);
            a1[i] = row_piece<T, ALIGNED>(wu, k, g.K, okf);
#pragma unroll
            for (int b = 0; b < MB; ++b) bx[i][b] = row_piece<T, ALIGNED>(xr[b], k, g.K, b * 16 + r < g.M);
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
        const int m = (e >> 6) * 16 + (e & 15);
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
// dst[row][0 .. ld): src row, zero from `cols` on
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(const T* src, long long s_ld, int rows, int cols, T* dst, int ld) {
    const long long total = (long long)rows * ld;
    for (long long o = (long long)blockIdx.x * 256 + threadIdx.x; o < total; o += 256ll * gridDim.x) {
        const int c = (int)(o % ld);
        dst[o] = c < cols ? src[(o / ld) * s_ld + c] : (T)0.f;
    }
}

// dst[c][at + r] = src[r][c]; columns at + rows .. at + ld_rows of dst are cleared
template <typename T>
__global__ __launch_bounds__(256) void transpose_kernel(const T* src, long long s_ld, int rows, int cols, T* dst, long long d_ld, int padded) {
    __shared__ T tile[64][65];
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
    for (int r = y; r < 64; r += 4) tile[r][x] = r0 + r < rows && c0 + x < cols ? src[(long long)(r0 + r) * s_ld + c0 + x] : (T)0.f;
    __syncthreads();
    for (int c = y; c < 64; c += 4)
        if (c0 + c < cols && r0 + x < padded) dst[(long long)(c0 + c) * d_ld + r0 + x] = tile[x][c];
}

// dG, dU from the saved projections: rows [M][2 Fp] (dG, then dU, each zero from F on) for the product with the weights, and
// transposed [2 F][Mp] (zero from M on) for the product with x.
template <typename T>
__global__ __launch_bounds__(256) void gate_slope_kernel(int M, int F, int Mp, int Fp, int act, const float* pre, const T* dh, long long dh_ld,
                                                         T* rows, T* cols) {
    __shared__ T tile[2][64][65];
    const int m0 = blockIdx.x * 64, f0 = blockIdx.y * 64, x = threadIdx.x & 63, y = threadIdx.x >> 6;
    const long long total = (long long)M * F;
    for (int r = y; r < 64; r += 4) {
        const int m = m0 + r, f = f0 + x;
        T vg = (T)0.f, vu = (T)0.f;
        if (m < M && f < F) {
            const long long o = (long long)m * F + f;
            const float d = (float)dh[(long long)m * dh_ld + f];
            const float2 a = activation(act, pre[o]);
            vg = (T)(d * pre[total + o] * a.y);
            vu = (T)(d * a.x);
        }
        if (m < M && f < Fp) {
            rows[(long long)m * 2 * Fp + f] = vg;
            rows[(long long)m * 2 * Fp + Fp + f] = vu;
        }
        tile[0][r][x] = vg;
        tile[1][r][x] = vu;
    }
    __syncthreads();
    for (int c = y; c < 64; c += 4)
        if (f0 + c < F && m0 + x < Mp) {
            cols[(long long)(f0 + c) * Mp + m0 + x] = tile[0][x][c];
            cols[(long long)(F + f0 + c) * Mp + m0 + x] = tile[1][x][c];
        }
}

static int ffn_check(const char* what, int dtype, int M, int K, int F, int act) {
    NMPC_REQUIRE(dtype >= NMPC_F32 && dtype <= NMPC_F16, "%s: unknown element type %d", what, dtype);
    NMPC_REQUIRE(M >= 0 && K >= 1 && F >= 1, "%s: bad sizes (%d rows, %d inputs, %d hidden units)", what, M, K, F);
    NMPC_REQUIRE(act >= NMPC_ACT_SILU && act <= NMPC_ACT_SIGMOID, "%s: activation %d", what, act);
    NMPC_REQUIRE(M < (1 << 22) && K < (1 << 21) && F < (1 << 21), "%s: at most 2^22 rows and 2^21 inputs and hidden units", what);
    return 0;
}
static unsigned long long round256(unsigned long long v) { return (v + 255) / 256 * 256; }

constexpr int FEW_ROWS = 64;

template <typename T>
constexpr int ktile() { return 128 / (int)sizeof(T); }
static int up_to(int v, int m) { return (v + m - 1) / m * m; }

// whether a matrix can be read in whole 128-byte k-tiles as it is
template <typename T>
static bool tiled(const void* p, long long ld, int K) {
    return K % ktile<T>() == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * sizeof(T) % 16 == 0;
}

// tile size and splits of a product: 256 x 256 where that gives the 256 CUs a tile each, else 128 x 128 (two workgroups a CU);
// the contraction is split where tiles alone leave CUs idle, into parts of at least 8 k-tiles
struct Shape {
    bool large;
    int splits;
};
static Shape product_shape(int M, int N, int ktiles, bool may_split) {
    const long long big = (long long)((M + 255) / 256) * ((N + 255) / 256), small = (long long)((M + 127) / 128) * ((N + 127) / 128);
    Shape s = {big >= 192, 1};
    if (!s.large && may_split && small < 256) {
        long long k = (512 + small - 1) / small;
        if (k > ktiles / 8) k = ktiles / 8;
        s.splits = k > 16 ? 16 : k < 1 ? 1 : (int)k;
    }
    return s;
}

template <typename T, bool GATED>
static int run_product(NtArgs g, hipStream_t st) {
    const int cols = GATED ? 2 * g.N : g.N;
    const Shape shape = product_shape(g.M, cols, g.ktiles, !GATED && g.part);
    g.splits = shape.splits;
    if (g.splits == 1) g.part = nullptr;
    const int bm = shape.large ? 256 : 128, bn = shape.large ? 256 : 128;
    g.mt = (g.M + bm - 1) / bm;
    g.nt = (g.N + (GATED ? bn / 2 : bn) - 1) / (GATED ? bn / 2 : bn);
    const long long grid = (long long)g.mt * g.nt * g.splits;
    NMPC_REQUIRE(grid < (1 << 22), "gated_ffn: too many tiles for one launch");
    if (shape.large) gemm_nt_kernel<T, 2, 4, 4, GATED><<<(unsigned)grid, 512, 0, st>>>(g);
    else gemm_nt_kernel<T, 2, 2, 2, GATED><<<(unsigned)grid, 256, 0, st>>>(g);
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

// The workspace of a call: copies of operands that cannot be read in k-tiles as they are, and the gradient's intermediates.
struct FfnSpace {
    unsigned long long bytes, x, wg, wu, rows, cols, wt, xt, part;
    template <typename T>
    static FfnSpace plan(int M, int K, int F, bool backward, bool copy) {
        FfnSpace s = {};
        const unsigned long long e = sizeof(T);
        const int kt = ktile<T>(), Kp = up_to(K, kt), Fp = up_to(F, kt), Mp = up_to(M, kt);
        auto take = [&](unsigned long long bytes) { const unsigned long long at = s.bytes; s.bytes += round256(bytes); return at; };
        if (!backward) {
            if (M > FEW_ROWS && (copy || K % kt)) {
                s.x = take(e * M * Kp);
                s.wg = take(e * F * Kp);
                s.wu = take(e * F * Kp);
            }
            return s;
        }
        s.rows = take(e * M * 2 * Fp);
        s.cols = take(e * 2 * F * Mp);
        s.wt = take(e * K * 2 * Fp);
        s.xt = take(e * K * Mp);
        const Shape a = product_shape(M, K, 2 * Fp / kt, true), b = product_shape(2 * F, K, Mp / kt, true);
        const unsigned long long pa = a.splits > 1 ? 4ull * a.splits * M * K : 0, pb = b.splits > 1 ? 4ull * b.splits * 2 * F * K : 0;
        s.part = take(pa > pb ? pa : pb);
        return s;
    }
};
template <typename T>
static bool needs_copy(int M, int K, const void* x, long long x_ld, const void* wg, const void* wu, long long w_ld) {
    return M > FEW_ROWS && !(tiled<T>(x, x_ld, K) && tiled<T>(wg, w_ld, K) && tiled<T>(wu, w_ld, K));
}

template <typename T>
static int run_forward(int M, int K, int F, const void* x, long long x_ld, const void* wg, const void* wu, long long w_ld, int act, void* h,
                       float* pre, char* ws, unsigned long long ws_bytes, hipStream_t st) {
    const bool copy = needs_copy<T>(M, K, x, x_ld, wg, wu, w_ld);
    const FfnSpace sp = FfnSpace::plan<T>(M, K, F, false, copy);
    NMPC_REQUIRE(sp.bytes == 0 || (ws && ws_bytes >= sp.bytes), "nmpc_gated_ffn: workspace of %llu bytes, %llu needed", ws_bytes, sp.bytes);
    if (M <= FEW_ROWS) {
        constexpr int E = 16 / sizeof(T);
        FewArgs g = {x, wg, wu, x_ld, w_ld, M, K, F, act, h, pre};
        const bool al = K % E == 0 && vec_ok<T>(x, x_ld, 0, E) && vec_ok<T>(wg, w_ld, 0, E) && vec_ok<T>(wu, w_ld, 0, E);
        const int blocks = (F + 15) / 16;
        int waves = 4;                 // enough waves to keep the memory busy: about 2048 on the chip
        while (waves < 16 && blocks * waves < 2048) waves *= 2;
        const int mb = M <= 16 ? 1 : M <= 32 ? 2 : 4;
        const unsigned shared = waves * 2 * mb * 64 * 16;
#define FEW(MB_)                                                                                                        \
    if (al) gated_few_kernel<T, MB_, true><<<blocks, waves * 64, shared, st>>>(g);                                      \
    else gated_few_kernel<T, MB_, false><<<blocks, waves * 64, shared, st>>>(g);
        if (mb == 1) { FEW(1) } else if (mb == 2) { FEW(2) } else {
            while (waves > 4) waves /= 2;
            const unsigned sh = waves * 2 * 4 * 64 * 16;
            if (al) gated_few_kernel<T, 4, true><<<blocks, waves * 64, sh, st>>>(g);
            else gated_few_kernel<T, 4, false><<<blocks, waves * 64, sh, st>>>(g);
        }
#undef FEW
        NMPC_HIP_CHECK(hipGetLastError());
        return 0;
    }
    NtArgs g = {};
    g.M = M; g.N = F; g.act = act; g.out = h; g.pre = pre; g.cut = M;
    const int Kp = up_to(K, ktile<T>());
    g.ktiles = Kp / ktile<T>();
    if (copy) {
        pad_kernel<T><<<pad_grid((long long)M * Kp), 256, 0, st>>>((const T*)x, x_ld, M, K, (T*)(ws + sp.x), Kp);
        pad_kernel<T><<<pad_grid((long long)F * Kp), 256, 0, st>>>((const T*)wg, w_ld, F, K, (T*)(ws + sp.wg), Kp);
        pad_kernel<T><<<pad_grid((long long)F * Kp), 256, 0, st>>>((const T*)wu, w_ld, F, K, (T*)(ws + sp.wu), Kp);
        x = ws + sp.x; wg = ws + sp.wg; wu = ws + sp.wu;
        x_ld = w_ld = Kp;
    }
    g.A = x; g.a_ld = x_ld; g.B = wg; g.B1 = wu; g.b_ld = w_ld;
    return run_product<T, true>(g, st);
}

template <typename T>
static int run_backward(int M, int K, int F, const void* x, long long x_ld, const void* wg, const void* wu, long long w_ld, int act,
                        const float* pre, const void* dh, long long dh_ld, void* dx, void* dwg, void* dwu, char* ws,
                        unsigned long long ws_bytes, hipStream_t st) {
    if (M == 0) {
        pad_kernel<T><<<pad_grid((long long)F * K), 256, 0, st>>>(nullptr, 0, F, 0, (T*)dwg, K);
        pad_kernel<T><<<pad_grid((long long)F * K), 256, 0, st>>>(nullptr, 0, F, 0, (T*)dwu, K);
        NMPC_HIP_CHECK(hipGetLastError());
        return 0;
    }
    const FfnSpace sp = FfnSpace::plan<T>(M, K, F, true, false);
    NMPC_REQUIRE(ws && ws_bytes >= sp.bytes, "nmpc_gated_ffn_bwd: workspace of %llu bytes, %llu needed", ws_bytes, sp.bytes);
    const int kt = ktile<T>(), Fp = up_to(F, kt), Mp = up_to(M, kt);
    T *rows = (T*)(ws + sp.rows), *cols = (T*)(ws + sp.cols), *wt = (T*)(ws + sp.wt), *xt = (T*)(ws + sp.xt);
    const int mb = (Mp + 63) / 64, kb = (K + 63) / 64, fb = (Fp + 63) / 64;
    gate_slope_kernel<T><<<dim3(mb, fb), 256, 0, st>>>(M, F, Mp, Fp, act, pre, (const T*)dh, dh_ld, rows, cols);
    transpose_kernel<T><<<dim3(fb, kb), 256, 0, st>>>((const T*)wg, w_ld, F, K, wt, 2 * Fp, Fp);
    transpose_kernel<T><<<dim3(fb, kb), 256, 0, st>>>((const T*)wu, w_ld, F, K, wt + Fp, 2 * Fp, Fp);
    transpose_kernel<T><<<dim3(mb, kb), 256, 0, st>>>((const T*)x, x_ld, M, K, xt, Mp, Mp);
    NtArgs g = {};
    g.A = rows; g.a_ld = 2 * Fp; g.B = wt; g.b_ld = 2 * Fp;
    g.M = M; g.N = K; g.ktiles = 2 * Fp / kt;
    g.out = dx; g.cut = M; g.part = (float*)(ws + sp.part);
    if (run_product<T, false>(g, st)) return 1;
    g.A = cols; g.a_ld = Mp; g.B = xt; g.b_ld = Mp;
    g.M = 2 * F; g.ktiles = Mp / kt;
    g.out = dwg; g.out1 = dwu; g.cut = F;
    return run_product<T, false>(g, st);
}

}  // namespace nmpc

using namespace nmpc;

extern "C" unsigned long long nmpc_gated_ffn_workspace_bytes(int dtype, int M, int K, int F, int backward, int copy) {
    if (M <= 0 || K <= 0 || F <= 0) return 0;
    return dtype == NMPC_F32 ? FfnSpace::plan<float>(M, K, F, backward != 0, copy != 0).bytes
                             : FfnSpace::plan<bf16>(M, K, F, backward != 0, copy != 0).bytes;
}

extern "C" int nmpc_gated_ffn(int dtype, int M, int K, int F, const void* x, long long x_ld, const void* wg, long long wg_ld,
                              const void* wu, long long wu_ld, int act, void* h, float* pre, void* workspace,
                              unsigned long long workspace_bytes, void* stream) {
    if (ffn_check("nmpc_gated_ffn", dtype, M, K, F, act)) return 1;
    if (M == 0) return 0;
    NMPC_REQUIRE(x && wg && wu && h, "nmpc_gated_ffn: null argument");
    NMPC_REQUIRE(wg_ld == wu_ld, "nmpc_gated_ffn: the weight matrices have different row strides");
    NMPC_DTYPE_SWITCH(dtype, { return run_forward<T_>(M, K, F, x, x_ld, wg, wu, wg_ld, act, h, pre, (char*)workspace, workspace_bytes, (hipStream_t)stream); })
    return 0;
}

extern "C" int nmpc_gated_ffn_bwd(int dtype, int M, int K, int F, const void* x, long long x_ld, const void* wg, long long wg_ld,
                                  const void* wu, long long wu_ld, int act, const float* pre, const void* dh, long long dh_ld, void* dx,
                                  void* dwg, void* dwu, void* workspace, unsigned long long workspace_bytes, void* stream) {
    if (ffn_check("nmpc_gated_ffn_bwd", dtype, M, K, F, act)) return 1;
    NMPC_REQUIRE(dwg && dwu && (M == 0 || (x && wg && wu && pre && dh && dx)), "nmpc_gated_ffn_bwd: null argument");
    NMPC_REQUIRE(wg_ld == wu_ld, "nmpc_gated_ffn_bwd: the weight matrices have different row strides");
    NMPC_DTYPE_SWITCH(dtype, { return run_backward<T_>(M, K, F, x, x_ld, wg, wu, wg_ld, act, pre, dh, dh_ld, dx, dwg, dwu, (char*)workspace, workspace_bytes, (hipStream_t)stream); })
    return 0;
}
