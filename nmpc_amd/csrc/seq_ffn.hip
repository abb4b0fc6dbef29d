// Gated feed-forward projections: h = act(x Wg') o (x Wu'), x[M,K], Wg / Wu[F,K], and their gradients
//   dG = dh o up o act'(gate),  dU = dh o act(gate),
//   dx = dG Wg + dU Wu,  dWg = dG' x,  dWu = dU' x.
// Both projections of a tile are accumulated side by side, so that the activation and the product happen in registers and
// neither projection is written (a training pass keeps both in fp32 for the gradient).  Products run on the matrix cores with
// fp32 accumulation; dG and dU are rounded to the element type once, as operands of the next products.
#include "seq_common.h"

namespace nmpc {

typedef float f32x4 __attribute__((ext_vector_type(4)));
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

// element (row, k) of an operand whose contraction index is split in two parts of `cut`
struct Operand {
    const void *p0, *p1;
    long long rs, ks;
};

struct GemmArgs {
    int M, N, K, act;                  // K: contraction of one part
    Operand A, B;
    int parts;                         // 1, 2: contraction over both parts
    void* out;                         // [M][N] (product) or h
    float* pre;                        // [2][M][N]: both projections (gated), may be null
};

template <typename T>
__device__ __forceinline__ f32x4 mfma_step(const T* a, const T* b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 mfma_step<bf16>(const bf16* a, const bf16* b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const bf16x8*)a, *(const bf16x8*)b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma_step<f16>(const f16* a, const f16* b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const f16x8*)a, *(const f16x8*)b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 mfma_step<float>(const float* a, const float* b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// 64 x 64 outputs of a block, 32 x 32 of a wave; GATED: B.p0 / B.p1 are the two weight matrices and both are accumulated.
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void gemm_kernel(GemmArgs g) {
    constexpr int BK = 32, LD = BK + 16 / sizeof(T), NB = GATED ? 2 : 1;
    __shared__ T sA[64][LD], sB[NB][64][LD];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    f32x4 acc[NB][2][2] = {};
    for (int part = 0; part < g.parts; ++part) {
        const T* A = (const T*)(part ? g.A.p1 : g.A.p0);
        const T* B[2] = {(const T*)(!GATED && part ? g.B.p1 : g.B.p0), (const T*)g.B.p1};
        for (int k0 = 0; k0 < g.K; k0 += BK) {
            __syncthreads();
            for (int e = tid; e < 64 * BK; e += 256) {
                // neighbouring threads along the contiguous axis
                const int ra = g.A.ks == 1 ? e / BK : e % 64, ka = g.A.ks == 1 ? e % BK : e / 64;
                const int rb = g.B.ks == 1 ? e / BK : e % 64, kb = g.B.ks == 1 ? e % BK : e / 64;
                sA[ra][ka] = m0 + ra < g.M && k0 + ka < g.K ? A[(m0 + ra) * g.A.rs + (k0 + ka) * g.A.ks] : (T)0.f;
#pragma unroll
                for (int i = 0; i < NB; ++i)
                    sB[i][rb][kb] = n0 + rb < g.N && k0 + kb < g.K ? B[i][(n0 + rb) * g.B.rs + (k0 + kb) * g.B.ks] : (T)0.f;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NB; ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        acc[i][r][c] = mfma_step<T>(&sA[wm + 16 * r + (lane & 15)][8 * (lane >> 4)], &sB[i][wn + 16 * c + (lane & 15)][8 * (lane >> 4)], acc[i][r][c]);
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int m = m0 + wm + 16 * r + 4 * (lane >> 4) + j, n = n0 + wn + 16 * c + (lane & 15);
                if (m >= g.M || n >= g.N) continue;
                const long long o = (long long)m * g.N + n;
                if constexpr (GATED) {
                    const float gate = acc[0][r][c][j], up = acc[NB - 1][r][c][j];
                    ((T*)g.out)[o] = (T)(activation(g.act, gate).x * up);
                    if (g.pre) { g.pre[o] = gate; g.pre[(long long)g.M * g.N + o] = up; }
                } else {
                    ((T*)g.out)[o] = (T)acc[0][r][c][j];
                }
            }
}

// dG, dU from the saved projections
template <typename T>
__global__ __launch_bounds__(256) void gate_slope_kernel(int M, int F, int act, const float* pre, const T* dh, long long dh_ld, T* dG, T* dU) {
    const long long total = (long long)M * F;
    for (long long o = (long long)blockIdx.x * 256 + threadIdx.x; o < total; o += 256ll * gridDim.x) {
        const float d = (float)dh[(o / F) * dh_ld + o % F];
        const float2 a = activation(act, pre[o]);
        dG[o] = (T)(d * pre[total + o] * a.y);
        dU[o] = (T)(d * a.x);
    }
}

static int ffn_check(const char* what, int dtype, int M, int K, int F, int act) {
    NMPC_REQUIRE(dtype >= NMPC_F32 && dtype <= NMPC_F16, "%s: unknown element type %d", what, dtype);
    NMPC_REQUIRE(M >= 0 && K >= 1 && F >= 1, "%s: bad sizes (%d rows, %d inputs, %d hidden units)", what, M, K, F);
    NMPC_REQUIRE(act >= NMPC_ACT_SILU && act <= NMPC_ACT_SIGMOID, "%s: activation %d", what, act);
    NMPC_REQUIRE(M < (1 << 22) && K < (1 << 22) && F < (1 << 22), "%s: sizes are below 2^22", what);
    return 0;
}
static unsigned long long round256(unsigned long long v) { return (v + 255) / 256 * 256; }

}  // namespace nmpc

using namespace nmpc;

extern "C" unsigned long long nmpc_gated_ffn_workspace_bytes(int dtype, int M, int K, int F, int backward) {
    if (M <= 0 || K <= 0 || F <= 0 || !backward) return 0;
    return 2 * round256((unsigned long long)M * F * (dtype == NMPC_F32 ? 4 : 2));
}

extern "C" int nmpc_gated_ffn(int dtype, int M, int K, int F, const void* x, long long x_ld, const void* wg, long long wg_ld,
                              const void* wu, long long wu_ld, int act, void* h, float* pre, void* workspace,
                              unsigned long long workspace_bytes, void* stream) {
    if (ffn_check("nmpc_gated_ffn", dtype, M, K, F, act)) return 1;
    if (M == 0) return 0;
    NMPC_REQUIRE(x && wg && wu && h, "nmpc_gated_ffn: null argument");
    NMPC_REQUIRE(wg_ld == wu_ld, "nmpc_gated_ffn: the weight matrices have different row strides");
    const unsigned long long need = nmpc_gated_ffn_workspace_bytes(dtype, M, K, F, 0);
    NMPC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "nmpc_gated_ffn: workspace of %llu bytes, %llu needed", workspace_bytes, need);
    GemmArgs g = {};
    g.M = M; g.N = F; g.K = K; g.act = act; g.parts = 1;
    g.A = {x, x, x_ld, 1};
    g.B = {wg, wu, wg_ld, 1};
    g.out = h; g.pre = pre;
    NMPC_DTYPE_SWITCH(dtype, { gemm_kernel<T_, true><<<dim3((F + 63) / 64, (M + 63) / 64), 256, 0, (hipStream_t)stream>>>(g); })
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int nmpc_gated_ffn_bwd(int dtype, int M, int K, int F, const void* x, long long x_ld, const void* wg, long long wg_ld,
                                  const void* wu, long long wu_ld, int act, const float* pre, const void* dh, long long dh_ld, void* dx,
                                  void* dwg, void* dwu, void* workspace, unsigned long long workspace_bytes, void* stream) {
    if (ffn_check("nmpc_gated_ffn_bwd", dtype, M, K, F, act)) return 1;
    NMPC_REQUIRE(dwg && dwu && (M == 0 || (x && wg && wu && pre && dh && dx)), "nmpc_gated_ffn_bwd: null argument");
    NMPC_REQUIRE(wg_ld == wu_ld, "nmpc_gated_ffn_bwd: the weight matrices have different row strides");
    const unsigned long long need = nmpc_gated_ffn_workspace_bytes(dtype, M, K, F, 1);
    NMPC_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "nmpc_gated_ffn_bwd: workspace of %llu bytes, %llu needed", workspace_bytes, need);
    const hipStream_t st = (hipStream_t)stream;
    NMPC_DTYPE_SWITCH(dtype, {
        T_* dG = (T_*)workspace;
        T_* dU = (T_*)((char*)workspace + need / 2);
        const long long total = (long long)M * F;
        if (M > 0) {
            gate_slope_kernel<T_><<<(unsigned)((total + 255) / 256 < (1 << 16) ? (total + 255) / 256 : (1 << 16)), 256, 0, st>>>(M, F, act, pre, (const T_*)dh, dh_ld, dG, dU);
            GemmArgs g = {};
            g.M = M; g.N = K; g.K = F; g.parts = 2;
            g.A = {dG, dU, F, 1};
            g.B = {wg, wu, 1, wg_ld};
            g.out = dx;
            gemm_kernel<T_, false><<<dim3((K + 63) / 64, (M + 63) / 64), 256, 0, st>>>(g);
        }
        for (int i = 0; i < 2; ++i) {
            GemmArgs g = {};
            g.M = F; g.N = K; g.K = M; g.parts = 1;
            g.A = {i ? dU : dG, nullptr, 1, F};
            g.B = {x, nullptr, 1, x_ld};
            g.out = i ? dwu : dwg;
            gemm_kernel<T_, false><<<dim3((K + 63) / 64, (F + 63) / 64), 256, 0, st>>>(g);
        }
    })
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}
