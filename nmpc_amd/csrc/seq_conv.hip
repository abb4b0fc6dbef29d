// Causal convolution over time, one short filter per channel, with an optional SiLU:
//   line = [start (W-1 rows); u],   s[t,c] = bias[c] + sum_j w[c,j] line[t+j,c],   y = act(s).
// Gradients, with ds = dy act'(s):
//   dline[k,c] = sum_j w[c,j] ds[k-j,c]  (+ dwindow where row k is one of the last W-1),   dw[c,j] = sum ds[t,c] line[t+j,c].
// All of it is bound by memory: one read of u and one write of y (backward: u, dy in, du out).  A thread owns a few neighbouring
// channels and a run of steps; the W-1 rows before the run (backward: behind it) are read again by the neighbouring run, mostly
// from the L2 cache, and everything else of the filter stays in registers.  Arithmetic and sums are fp32.
// Measured at bf16 4 x 2048 x 4096, W = 4.  Channels of a thread: forward 8 bytes 28 us (4.8 TB/s; 16 bytes 37 us: half the waves),
// backward 4 bytes 48 us (4.2 TB/s; 8 bytes 61 us).  Steps of a run: forward 16 (24 .. 28 us for 16 .. 32), backward 28 (16: 58 us,
// 24: 48, 32: 63; over ten shapes 28 is the least in seven): runs of 2^n rows of 2^m bytes meet on the same memory channels.
#include <type_traits>

#include "seq_common.h"

namespace nmpc {

constexpr int CONV_MAX_W = 8;
constexpr int CONV_TR = 16;          // steps of one thread, forward
constexpr int CONV_TR_BWD = 28;      // backward
constexpr int CONV_GROUP = 4;        // steps whose loads are in flight together

struct ConvArgs {
    int nb, L, D, silu, nch, ncv;
    const void* u;
    long long u_bs, u_ts;
    const float *w, *bias;
    const void* start;
    const int* lengths;
    void *y, *window;
    const void* dy;                  // backward
    long long dy_bs, dy_ts;
    const void* dwindow;
    void *du, *dstart;
    float* part;                     // [row blocks][W + 1][D] partial sums of dw, dbias
    int cvb, nrb;
};

// line[k] of sequence b, k = 0 .. W-2+L
template <typename T, int W, int VEC>
__device__ __forceinline__ Vec<T, VEC> line_row(const T* ub, long long u_ts, const T* sb, int D, int k) {
    if (k >= W - 1) return load_vec<T, VEC>(ub + (long long)(k - (W - 1)) * u_ts);
    if (sb) return load_vec<T, VEC>(sb + (long long)k * D);
    Vec<T, VEC> z;
#pragma unroll
    for (int i = 0; i < VEC; ++i) z.v[i] = (T)0.f;
    return z;
}

// f with the flag as a constant, so that the steps of a run are one block of code
template <typename F>
__device__ __forceinline__ void either(bool flag, F f) {
    if (flag) f(std::true_type{});
    else f(std::false_type{});
}

template <typename T, int W, int VEC>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvArgs a) {
    const unsigned gid = blockIdx.x * 256u + threadIdx.x;
    const unsigned row = gid / (unsigned)a.ncv;
    const int c = (int)(gid % (unsigned)a.ncv) * VEC;
    const int b = (int)(row / (unsigned)a.nch), t0 = (int)(row % (unsigned)a.nch) * CONV_TR;
    if (b >= a.nb) return;
    const int len = seq_length(a.lengths, b, a.L);
    const T* ub = (const T*)a.u + b * a.u_bs + c;
    const T* sb = a.start ? (const T*)a.start + (long long)b * (W - 1) * a.D + c : nullptr;
    T* yb = (T*)a.y + (long long)b * a.L * a.D + c;
    float w[W][VEC], bias[VEC], win[W][VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][i] = a.w[(long long)(c + i) * W + j];
        bias[i] = a.bias ? a.bias[c + i] : 0.f;
    }
    const int t1 = min(t0 + CONV_TR, a.L), tv = min(t1, len);
    if (t0 < tv) {
#pragma unroll
        for (int j = 0; j < W - 1; ++j) {
            const Vec<T, VEC> r = line_row<T, W, VEC>(ub, a.u_ts, sb, a.D, t0 + j);
#pragma unroll
            for (int i = 0; i < VEC; ++i) win[j][i] = (float)r.v[i];
        }
    }
    // rows of the run: a thread's own address plus multiples of the stride that are the same for all threads
    const T* ur = ub + t0 * a.u_ts;
    T* yr = yb + (long long)t0 * a.D;
    // all loads of a group of steps before its first store (the compiler cannot know that y is not u)
    auto group = [&](int k0, auto whole, auto silu) {
        Vec<T, VEC> rows[CONV_GROUP];
#pragma unroll
        for (int k = 0; k < CONV_GROUP; ++k)
            if (whole.value || t0 + k0 + k < tv) rows[k] = load_vec<T, VEC>(ur + (k0 + k) * a.u_ts);
#pragma unroll
        for (int k = 0; k < CONV_GROUP; ++k) {
            if (!whole.value && t0 + k0 + k >= tv) break;
            Vec<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                win[W - 1][i] = (float)rows[k].v[i];
                float s = bias[i];
#pragma unroll
                for (int j = 0; j < W; ++j) s += w[j][i] * win[j][i];
                o.v[i] = (T)(silu.value ? s * sigmoid(s) : s);
#pragma unroll
                for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
            }
            store_vec(yr + (long long)(k0 + k) * a.D, o);
        }
    };
    either(a.silu, [&](auto silu) {
        if (tv == t0 + CONV_TR) {
#pragma unroll
            for (int k = 0; k < CONV_TR; k += CONV_GROUP) group(k, std::true_type{}, silu);
        } else {
            for (int k = 0; t0 + k < tv; k += CONV_GROUP) group(k, std::false_type{}, silu);
        }
    });
    Vec<T, VEC> zero;
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero.v[i] = (T)0.f;
    for (int t = max(t0, tv); t < t1; ++t) store_vec(yb + (long long)t * a.D, zero);
    if (a.window && t0 == 0) {                     // the last W-1 rows of the line, bit for bit
        T* ob = (T*)a.window + (long long)b * (W - 1) * a.D + c;
#pragma unroll
        for (int j = 0; j < W - 1; ++j) store_vec(ob + (long long)j * a.D, line_row<T, W, VEC>(ub, a.u_ts, sb, a.D, len + j));
    }
}

// ds of step t and the step's row of u; `win` holds the W-1 rows before it and is shifted
template <typename T, int W, int VEC>
__device__ __forceinline__ void conv_slope(bool silu, const Vec<T, VEC>& r, const Vec<T, VEC>& g, const float (&w)[W][VEC],
                                           const float (&bias)[VEC], float (&win)[W][VEC], float (&ds)[VEC]) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        win[W - 1][i] = (float)r.v[i];
        float s = bias[i];
#pragma unroll
        for (int j = 0; j < W; ++j) s += w[j][i] * win[j][i];
        float k = (float)g.v[i];
        if (silu) {
            const float p = sigmoid(s);
            k *= p * (1.f + s * (1.f - p));
        }
        ds[i] = k;
    }
}

// A block holds cvb channel vectors x (256 / cvb) runs; the runs' sums for dw and dbias are joined through LDS in run order.
template <typename T, int W, int VEC>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvArgs a) {
    __shared__ float red[VEC][256];
    const int tid = threadIdx.x, rows = 256 / a.cvb;
    const int cb = (int)(blockIdx.x % ((a.ncv + a.cvb - 1) / a.cvb)), rb = (int)(blockIdx.x / ((a.ncv + a.cvb - 1) / a.cvb));
    const int cv = cb * a.cvb + tid % a.cvb;
    const long long row = (long long)rb * rows + tid / a.cvb;
    const int c = cv * VEC;
    const int b = (int)(row / a.nch), t0 = (int)(row % a.nch) * CONV_TR_BWD;
    float dw[W + 1][VEC];
#pragma unroll
    for (int j = 0; j <= W; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) dw[j][i] = 0.f;
    if (cv < a.ncv && b < a.nb) {
        const int len = seq_length(a.lengths, b, a.L);
        const T* ub = (const T*)a.u + b * a.u_bs + c;
        const T* gb = (const T*)a.dy + b * a.dy_bs + c;
        const T* sb = a.start ? (const T*)a.start + (long long)b * (W - 1) * a.D + c : nullptr;
        const T* eb = a.dwindow ? (const T*)a.dwindow + (long long)b * (W - 1) * a.D + c : nullptr;
        T* db = (T*)a.du + (long long)b * a.L * a.D + c;
        float w[W][VEC], bias[VEC], win[W][VEC], ds[W][VEC];      // ds[i]: steps t-W+1+i
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) w[j][i] = a.w[(long long)(c + i) * W + j];
            bias[i] = a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
            for (int j = 0; j < W; ++j) ds[j][i] = 0.f;
        }
        const int t1 = min(t0 + CONV_TR_BWD, a.L), tv = min(t1, len);
        if (t0 < tv) {
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                const Vec<T, VEC> r = line_row<T, W, VEC>(ub, a.u_ts, sb, a.D, t0 + j);
#pragma unroll
                for (int i = 0; i < VEC; ++i) win[j][i] = (float)r.v[i];
            }
        }
        // row k of the line's gradient is complete once ds of steps k-W+1 .. k is known
        const int tl = min(tv + W - 1, len);           // steps that are read
        // the run's rows, one after the other: sums instead of products of 64 bits in every lane and access
        const T* ur = ub + t0 * a.u_ts;
        const T* gr = gb + t0 * a.dy_ts;
        T* dr = db + (long long)t0 * a.D;
        // step k of the run; whole: all W - 1 steps behind the run are inside the sequence, so that only k decides
        auto step = [&](int k, const Vec<T, VEC>& ru, const Vec<T, VEC>& rg, auto whole, auto silu) {
            const int t = t0 + k;
            if (whole.value || t < tl) {
                conv_slope<T, W, VEC>(silu.value, ru, rg, w, bias, win, ds[W - 1]);
                if (whole.value ? k < CONV_TR_BWD : t < tv) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
#pragma unroll
                        for (int j = 0; j < W; ++j) dw[j][i] += ds[W - 1][i] * win[j][i];
                        dw[W][i] += ds[W - 1][i];
                        // (added here: put off to the end, they would keep every step's ds and win in registers)
#pragma unroll
                        for (int j = 0; j <= W; ++j) asm volatile("" : "+v"(dw[j][i]));
                    }
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i)
#pragma unroll
                    for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) ds[W - 1][i] = 0.f;
            }
            if (k >= W - 1) {                          // u[t - W + 1] is row t of the line; it feeds steps t - W + 1 .. t
                Vec<T, VEC> o, e;
                const bool end = !whole.value && eb && t >= len;
                if (end) e = load_vec<T, VEC>(eb + (long long)(t - len) * a.D);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float v = end ? (float)e.v[i] : 0.f;
#pragma unroll
                    for (int j = 0; j < W; ++j) v += w[W - 1 - j][i] * ds[j][i];
                    o.v[i] = (T)v;
                }
                store_vec(dr, o);
                dr += a.D;
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i)
#pragma unroll
                for (int j = 0; j < W - 1; ++j) ds[j][i] = ds[j + 1][i];
        };
        either(a.silu, [&](auto silu) {
            if (tv == t0 + CONV_TR_BWD && tl == tv + W - 1) {
                constexpr int STEPS = CONV_TR_BWD + W - 1;
                Vec<T, VEC> ru[2][CONV_GROUP], rg[2][CONV_GROUP];      // the next group's rows are loaded while this one's are used
                auto fetch = [&](int g) {
#pragma unroll
                    for (int k = 0; k < CONV_GROUP; ++k)
                        if (g * CONV_GROUP + k < STEPS) {
                            ru[g & 1][k] = load_vec<T, VEC>(ur);
                            rg[g & 1][k] = load_vec<T, VEC>(gr);
                            ur += a.u_ts;
                            gr += a.dy_ts;
                        }
                };
                fetch(0);
#pragma unroll
                for (int g = 0; g * CONV_GROUP < STEPS; ++g) {
                    if ((g + 1) * CONV_GROUP < STEPS) fetch(g + 1);
#pragma unroll
                    for (int k = 0; k < CONV_GROUP; ++k)
                        if (g * CONV_GROUP + k < STEPS) step(g * CONV_GROUP + k, ru[g & 1][k], rg[g & 1][k], std::true_type{}, silu);
                }
            } else {
                for (int k = 0; t0 + k < tv + W - 1; ++k) {
                    Vec<T, VEC> ru, rg;
                    if (t0 + k < tl) {
                        ru = load_vec<T, VEC>(ur);
                        rg = load_vec<T, VEC>(gr);
                        ur += a.u_ts;
                        gr += a.dy_ts;
                    }
                    step(k, ru, rg, std::false_type{}, silu);
                }
            }
        });
        Vec<T, VEC> zero;
#pragma unroll
        for (int i = 0; i < VEC; ++i) zero.v[i] = (T)0.f;
        for (int t = max(t0, tv); t < t1; ++t) store_vec(db + (long long)t * a.D, zero);
        if (a.dstart && t0 == 0) {                     // rows k < W-1 of the line feed steps 0 .. k
            T* ob = (T*)a.dstart + (long long)b * (W - 1) * a.D + c;
            float head[W][VEC];
#pragma unroll
            for (int j = 0; j < W - 1; ++j) {
                const Vec<T, VEC> r = line_row<T, W, VEC>(ub, a.u_ts, sb, a.D, j);
#pragma unroll
                for (int i = 0; i < VEC; ++i) { win[j][i] = (float)r.v[i]; head[j][i] = 0.f; }
            }
#pragma unroll
            for (int t = 0; t < W - 1; ++t)
                if (t < len) {
                    conv_slope<T, W, VEC>(a.silu, load_vec<T, VEC>(ub + t * a.u_ts), load_vec<T, VEC>(gb + t * a.dy_ts), w, bias, win, ds[0]);
#pragma unroll
                    for (int k = t; k < W - 1; ++k)
#pragma unroll
                        for (int i = 0; i < VEC; ++i) head[k][i] += w[k - t][i] * ds[0][i];
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
#pragma unroll
                        for (int j = 0; j < W - 1; ++j) win[j][i] = win[j + 1][i];
                }
#pragma unroll
            for (int k = 0; k < W - 1; ++k) {
                Vec<T, VEC> o, e;
                if (eb && k >= len) e = load_vec<T, VEC>(eb + (long long)(k - len) * a.D);
#pragma unroll
                for (int i = 0; i < VEC; ++i) o.v[i] = (T)(head[k][i] + (eb && k >= len ? (float)e.v[i] : 0.f));
                store_vec(ob + (long long)k * a.D, o);
            }
        }
    }
    if (a.nrb == 0) return;                            // no steps at all: dw and dbias are zero
#pragma unroll
    for (int j = 0; j <= W; ++j) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VEC; ++i) red[i][tid] = dw[j][i];
        __syncthreads();
        for (int e = tid; e < a.cvb * VEC; e += 256) {
            const int ch = cb * a.cvb * VEC + e;
            float s = 0.f;
            for (int r = 0; r < rows; ++r) s += red[e % VEC][r * a.cvb + e / VEC];
            if (ch < a.D) a.part[((long long)rb * (W + 1) + j) * a.D + ch] = s;
        }
    }
}

// dw[c][j], dbias[c]: sums of the row blocks' partial sums, always in the same order
__global__ __launch_bounds__(256) void conv_reduce_kernel(const float* part, int nrb, int W, int D, float* dw, float* dbias) {
    __shared__ float red[256];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), sub = threadIdx.x >> 6, j = blockIdx.y;
    float s = 0.f;
    if (c < D)
        for (int r = sub; r < nrb; r += 4) s += part[((long long)r * (W + 1) + j) * D + c];
    red[threadIdx.x] = s;
    __syncthreads();
    if (sub == 0 && c < D) {
        s = (red[threadIdx.x] + red[threadIdx.x + 64]) + (red[threadIdx.x + 128] + red[threadIdx.x + 192]);
        if (j < W) dw[(long long)c * W + j] = s;
        else if (dbias) dbias[c] = s;
    }
}

// One step of every sequence: the window moves on by one row in place.
template <typename T, int W, int VEC>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvArgs a) {
    const unsigned gid = blockIdx.x * 256u + threadIdx.x;
    const int b = (int)(gid / (unsigned)a.ncv), c = (int)(gid % (unsigned)a.ncv) * VEC;
    if (b >= a.nb) return;
    T* wb = (T*)a.window + (long long)b * (W - 1) * a.D + c;
    Vec<T, VEC> line[W], o;
#pragma unroll
    for (int j = 0; j < W - 1; ++j) line[j] = load_vec<T, VEC>(wb + (long long)j * a.D);
    line[W - 1] = load_vec<T, VEC>((const T*)a.u + b * a.u_bs + c);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        float s = a.bias ? a.bias[c + i] : 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) s += a.w[(long long)(c + i) * W + j] * (float)line[j].v[i];
        o.v[i] = (T)(a.silu ? s * sigmoid(s) : s);
    }
#pragma unroll
    for (int j = 0; j < W - 1; ++j) store_vec(wb + (long long)j * a.D, line[j + 1]);
    store_vec((T*)a.y + (long long)b * a.D + c, o);
}

// rows (runs) of a backward block and the number of blocks of rows; VEC only changes how many channels a vector has
inline int conv_cvb(int ncv) {
    int v = 1;
    while (v < ncv && v < 32) v *= 2;
    return v;
}
inline int conv_nch(int L, int run) { return L > run ? (L + run - 1) / run : 1; }

#define NMPC_W_SWITCH(W, ...)                                                                                      \
    switch (W) {                                                                                                   \
        case 1: { constexpr int W_ = 1; __VA_ARGS__ } break; case 2: { constexpr int W_ = 2; __VA_ARGS__ } break;                \
        case 3: { constexpr int W_ = 3; __VA_ARGS__ } break; case 4: { constexpr int W_ = 4; __VA_ARGS__ } break;                \
        case 5: { constexpr int W_ = 5; __VA_ARGS__ } break; case 6: { constexpr int W_ = 6; __VA_ARGS__ } break;                \
        case 7: { constexpr int W_ = 7; __VA_ARGS__ } break; case 8: { constexpr int W_ = 8; __VA_ARGS__ } break;                \
        default: set_error("causal_conv: %d taps (1..8)", W); return 1;                                           \
    }

static int conv_check(const char* what, int nb, int L, int D, int W, int act) {
    NMPC_REQUIRE(nb >= 0 && L >= 0 && D >= 1, "%s: bad sizes (%d sequences, %d steps, %d channels)", what, nb, L, D);
    NMPC_REQUIRE(W >= 1 && W <= CONV_MAX_W, "%s: %d taps (1..%d)", what, W, CONV_MAX_W);
    NMPC_REQUIRE(D < 1 << 30, "%s: %d channels (fewer than 2^30)", what, D);       // the sums of dw: four threads a channel, fewer than 2^32 a launch
    NMPC_REQUIRE(act == NMPC_ACT_NONE || act == NMPC_ACT_SILU, "%s: activation %d (none or silu)", what, act);
    NMPC_REQUIRE(L <= 1 << 30, "%s: at most 2^30 steps", what);
    NMPC_REQUIRE((long long)nb * conv_nch(L, CONV_TR) * D < (1ll << 31), "%s: too many elements for one launch", what);
    return 0;
}

}  // namespace nmpc

using namespace nmpc;

extern "C" int nmpc_causal_conv(int dtype, int nb, int L, int D, int W, const void* u, long long u_bs, long long u_ts,
                                const float* w, const float* bias, int act, const void* start, const int* lengths, void* y,
                                void* window, void* stream) {
    if (conv_check("nmpc_causal_conv", nb, L, D, W, act)) return 1;
    if (nb == 0) return 0;
    NMPC_REQUIRE(w && (L == 0 || (u && y)), "nmpc_causal_conv: null argument");
    ConvArgs a = {};
    a.nb = nb; a.L = L; a.D = D; a.silu = act == NMPC_ACT_SILU; a.nch = conv_nch(L, CONV_TR);
    a.u = u; a.u_bs = u_bs; a.u_ts = u_ts; a.w = w; a.bias = bias; a.start = start; a.lengths = lengths;
    a.y = y; a.window = W > 1 ? window : nullptr;
    NMPC_DTYPE_SWITCH(dtype, {
        constexpr int V = 8 / sizeof(T_);
        const bool vec = D % V == 0 && vec_ok<T_>(u, u_bs, u_ts, V) && vec_ok<T_>(start, 0, 0, V) && vec_ok<T_>(y, 0, 0, V) &&
                         vec_ok<T_>(window, 0, 0, V);
        a.ncv = vec ? D / V : D;
        const unsigned grid = (unsigned)(((long long)nb * a.nch * a.ncv + 255) / 256);
        NMPC_W_SWITCH(W, {
            if (vec) conv_fwd_kernel<T_, W_, V><<<grid, 256, 0, (hipStream_t)stream>>>(a);
            else conv_fwd_kernel<T_, W_, 1><<<grid, 256, 0, (hipStream_t)stream>>>(a);
        })
    })
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" unsigned long long nmpc_causal_conv_workspace_bytes(int nb, int L, int D, int W) {
    if (nb <= 0 || L <= 0 || D <= 0 || W <= 0) return 0;
    // fewest runs a block can hold: 8, with 32 channel vectors
    const unsigned long long nrb = ((unsigned long long)nb * conv_nch(L, CONV_TR_BWD) + 7) / 8;
    return nrb * (W + 1) * D * sizeof(float);
}

extern "C" int nmpc_causal_conv_bwd(int dtype, int nb, int L, int D, int W, const void* u, long long u_bs, long long u_ts,
                                    const float* w, const float* bias, int act, const void* start, const int* lengths,
                                    const void* dy, long long dy_bs, long long dy_ts, const void* dwindow, void* du, float* dw,
                                    float* dbias, void* dstart, void* workspace, unsigned long long workspace_bytes, void* stream) {
    if (conv_check("nmpc_causal_conv_bwd", nb, L, D, W, act)) return 1;
    NMPC_REQUIRE(w && dw && (nb == 0 || L == 0 || (u && dy && du)), "nmpc_causal_conv_bwd: null argument");
    NMPC_REQUIRE(workspace_bytes >= nmpc_causal_conv_workspace_bytes(nb, L, D, W), "nmpc_causal_conv_bwd: workspace of %llu bytes, %llu needed",
                 workspace_bytes, nmpc_causal_conv_workspace_bytes(nb, L, D, W));
    NMPC_REQUIRE(workspace || nb == 0 || L == 0, "nmpc_causal_conv_bwd: null workspace");
    ConvArgs a = {};
    a.nb = nb; a.L = L; a.D = D; a.silu = act == NMPC_ACT_SILU; a.nch = conv_nch(L, CONV_TR_BWD);
    a.u = u; a.u_bs = u_bs; a.u_ts = u_ts; a.w = w; a.bias = bias; a.start = start; a.lengths = lengths;
    a.dy = dy; a.dy_bs = dy_bs; a.dy_ts = dy_ts; a.dwindow = W > 1 ? dwindow : nullptr; a.du = du; a.dstart = W > 1 ? dstart : nullptr;
    a.part = (float*)workspace;
    a.nrb = 0;
    if (nb > 0 && (L > 0 || a.dstart)) {
        NMPC_DTYPE_SWITCH(dtype, {
            constexpr int V = 4 / sizeof(T_);
            const bool vec = D % V == 0 && vec_ok<T_>(u, u_bs, u_ts, V) && vec_ok<T_>(start, 0, 0, V) && vec_ok<T_>(dy, dy_bs, dy_ts, V) &&
                             vec_ok<T_>(dwindow, 0, 0, V) && vec_ok<T_>(du, 0, 0, V) && vec_ok<T_>(dstart, 0, 0, V);
            a.ncv = vec ? D / V : D;
            a.cvb = conv_cvb(a.ncv);
            const int rows = 256 / a.cvb;
            const long long nrb = ((long long)nb * a.nch + rows - 1) / rows;
            a.nrb = L > 0 ? (int)nrb : 0;
            const unsigned grid = (unsigned)(nrb * ((a.ncv + a.cvb - 1) / a.cvb));
            NMPC_W_SWITCH(W, {
                if (vec) conv_bwd_kernel<T_, W_, V><<<grid, 256, 0, (hipStream_t)stream>>>(a);
                else conv_bwd_kernel<T_, W_, 1><<<grid, 256, 0, (hipStream_t)stream>>>(a);
            })
        })
        NMPC_HIP_CHECK(hipGetLastError());
    }
    conv_reduce_kernel<<<dim3((D + 63) / 64, W + 1), 256, 0, (hipStream_t)stream>>>(a.part, a.nrb, W, D, dw, dbias);
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}

extern "C" int nmpc_causal_conv_step(int dtype, int nb, int D, int W, void* window, const void* u, long long u_bs, const float* w,
                                     const float* bias, int act, void* y, void* stream) {
    if (conv_check("nmpc_causal_conv_step", nb, 1, D, W, act)) return 1;
    if (nb == 0) return 0;
    NMPC_REQUIRE(u && w && y && (window || W == 1), "nmpc_causal_conv_step: null argument");
    ConvArgs a = {};
    a.nb = nb; a.L = 1; a.D = D; a.silu = act == NMPC_ACT_SILU;
    a.u = u; a.u_bs = u_bs; a.w = w; a.bias = bias; a.y = y; a.window = window;
    NMPC_DTYPE_SWITCH(dtype, {
        constexpr int V = 8 / sizeof(T_);
        const bool vec = D % V == 0 && vec_ok<T_>(u, u_bs, 0, V) && vec_ok<T_>(y, 0, 0, V) && vec_ok<T_>(window, 0, 0, V);
        a.ncv = vec ? D / V : D;
        const unsigned grid = (unsigned)(((long long)nb * a.ncv + 255) / 256);
        NMPC_W_SWITCH(W, {
            if (vec) conv_step_kernel<T_, W_, V><<<grid, 256, 0, (hipStream_t)stream>>>(a);
            else conv_step_kernel<T_, W_, 1><<<grid, 256, 0, (hipStream_t)stream>>>(a);
        })
    })
    NMPC_HIP_CHECK(hipGetLastError());
    return 0;
}
