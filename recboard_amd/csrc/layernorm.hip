// Layer norm over the last dimension, alone or behind a residual sum, forward and backward (fp32, bf16, fp16).
//
//   s = x + r (r optional),  mean = sum s / D,  var = sum (s - mean)^2 / D,  rstd = 1 / sqrt(var + eps),  y = (s - mean) rstd w + b
//   backward, g = dy w, xhat = (s - mean) rstd:   ds' = rstd (g - mean(g) - xhat mean(g xhat)) + ds,  dw = sum_rows dy xhat,  db = sum_rows dy
//
// Both passes are bound by HBM: a row is read once and stays in registers, so the variance is the sum of squared deviations from the finished
// mean (two passes over registers, not over memory, and no cancellation of a sum of squares against a squared sum).  LPR lanes share a row
// (a part of a wave for narrow rows, a wave, or a workgroup of 256 - 1024 lanes), each with N pieces of VEC consecutive elements (16
// bytes; rows that start anywhere are read the same way, their last piece element by element).
// The backward's column sums stay in the registers of the lanes that own the columns over all rows of a workgroup; one partial row of dw and
// one of db per workgroup go to the workspace and a second launch adds them in a fixed order (no atomics: run to run the same bits).
// Measured: 16384 x 4096 bf16 behind a residual: forward 96 - 105 us (537 MB: 5.1 - 5.6 TB/s), backward 120 + 5 us (4.5 TB/s); a copy reaches 4.9.
// All statistics and sums are fp32; s is rounded to the tensor's type once, for the store, while y comes from the unrounded sum.  The backward reads that
// rounded s with the mean and rstd of the unrounded one (x and r again would be a fifth stream of HBM for four): xhat, and dw with it, is off by
// up to u |s| / std of its row, u = 2^-8 (bf16) or 2^-11 (fp16): rows whose mean is far larger than their spread lose that much there.
#include "re_types.h"

namespace {

constexpr int LN_MAX_D = 1 << 24;

struct ln_args {
    const void *x, *r, *w, *b;
    void *y, *s;
    float *mean, *rstd;
    int64_t rows;
    int32_t D, wtype;
    float eps;
};
struct ln_bwd_args {
    const void *dy, *s, *w, *ds;
    void* dx;
    const float *mean, *rstd;
    float* part;      // [gridDim.x][2][D]
    int64_t rows;
    int32_t D, wtype;
};

// sum over the LPR lanes of a row; every lane of the row gets it.  `red` : 2 * 16 floats of LDS (rows wider than a wave)
template <int LPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    constexpr int W = LPR < 64 ? LPR : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if constexpr (LPR > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();                       // the previous sum has been read
        if ((threadIdx.x & 63) == 0) red[wave] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < LPR / 64; ++i) v += red[i];
    }
    return v;
}
template <int LPR>
__device__ __forceinline__ void row_sum2(float& a, float& c, float* red) {
    constexpr int W = LPR < 64 ? LPR : 64;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
        a += __shfl_xor(a, o, 64);
        c += __shfl_xor(c, o, 64);
    }
    if constexpr (LPR > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) {
            red[wave] = a;
            red[16 + wave] = c;
        }
        __syncthreads();
        a = c = 0.f;
#pragma unroll
        for (int i = 0; i < LPR / 64; ++i) {
            a += red[i];
            c += red[16 + i];
        }
    }
}

// the lane's pieces of a weight (null: `none` everywhere; beyond D: 0).  Of the tensor's own type, the usual case, by 16-byte pieces; of another
// element by element (a served token's row is its weights' latency: 7.8 us for one row of 4096 with the element loads, all types).
template <class T, int LPR, int VEC, int N>
__device__ __forceinline__ void load_weight(const void* w, int32_t wtype, int D, int lane, float none, float* f) {
    if (!w) {
#pragma unroll
        for (int i = 0; i < N * VEC; ++i) f[i] = none;
    } else if (wtype == re_type<T>::CODE) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = (n * LPR + lane) * VEC;
            if (e < D) {
                re_load_some<T, VEC, false>(static_cast<const T*>(w) + e, D - e, f + n * VEC);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) f[n * VEC + v] = 0.f;
            }
        }
    } else {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int e = (n * LPR + lane) * VEC + v;
                f[n * VEC + v] = e < D ? re_load_as_float(w, e, wtype) : 0.f;
            }
    }
}

template <class T, int LPR, int VEC, int N, bool ALIGNED>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void ln_fwd_k(const ln_args a) {
    constexpr int THREADS = LPR > 256 ? LPR : 256, RPW = THREADS / LPR;
    __shared__ float red[32];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const int D = a.D;
    float w[N * VEC], b[N * VEC];
    load_weight<T, LPR, VEC, N>(a.w, a.wtype, D, lane, 1.f, w);
    load_weight<T, LPR, VEC, N>(a.b, a.wtype, D, lane, 0.f, b);
    const float inv_d = 1.f / (float)D;
    const int64_t steps = (a.rows + RPW - 1) / RPW;
    for (int64_t step = blockIdx.x; step < steps; step += gridDim.x) {
        const int64_t row = step * RPW + sub;
        const bool live = row < a.rows;
        const T* x = static_cast<const T*>(a.x) + row * D;
        const T* r = a.r ? static_cast<const T*>(a.r) + row * D : nullptr;
        float f[N * VEC];
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = (n * LPR + lane) * VEC;
            if (live && e < D) {
                re_load_some<T, VEC, ALIGNED>(x + e, D - e, f + n * VEC);
                if (r) {
                    float g[VEC];
                    re_load_some<T, VEC, ALIGNED>(r + e, D - e, g);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) f[n * VEC + v] += g[v];
                }
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) f[n * VEC + v] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < N * VEC; ++i) sum += f[i];
        const float mean = row_sum<LPR>(sum, red) * inv_d;
        float sq = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = (n * LPR + lane) * VEC;
            if (e < D) {
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float d = f[n * VEC + v] - mean;
                    if (ALIGNED || e + v < D) sq += d * d;
                }
            }
        }
        const float rstd = 1.f / sqrtf(row_sum<LPR>(sq, red) * inv_d + a.eps);
        if (live) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int e = (n * LPR + lane) * VEC;
                if (e < D) {
                    float o[VEC];
#pragma unroll
                    for (int v = 0; v < VEC; ++v) o[v] = (f[n * VEC + v] - mean) * rstd * w[n * VEC + v] + b[n * VEC + v];
                    re_store_some<T, VEC, ALIGNED>(static_cast<T*>(a.y) + row * D + e, D - e, o);
                    if (a.s) re_store_some<T, VEC, ALIGNED>(static_cast<T*>(a.s) + row * D + e, D - e, f + n * VEC);
                }
            }
            if (lane == 0) {
                if (a.mean) a.mean[row] = mean;
                if (a.rstd) a.rstd[row] = rstd;
            }
        }
    }
}

// The backward of the rows and this workgroup's part of the column sums.
template <class T, int LPR, int VEC, int N, bool ALIGNED>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void ln_bwd_k(const ln_bwd_args a) {
    constexpr int THREADS = LPR > 256 ? LPR : 256, RPW = THREADS / LPR;
    constexpr int COLS = LPR * VEC * N;                      // columns that the lanes of a row own
    __shared__ float red[32];
    __shared__ float join[LPR < 256 ? (LPR < 64 ? 4 : RPW) * COLS : 1];
    const int lane = threadIdx.x % LPR, sub = threadIdx.x / LPR;
    const int D = a.D;
    float w[N * VEC], dw[N * VEC], db[N * VEC];
    load_weight<T, LPR, VEC, N>(a.w, a.wtype, D, lane, 1.f, w);
#pragma unroll
    for (int i = 0; i < N * VEC; ++i) dw[i] = db[i] = 0.f;
    const float inv_d = 1.f / (float)D;
    const int64_t steps = (a.rows + RPW - 1) / RPW;
    for (int64_t step = blockIdx.x; step < steps; step += gridDim.x) {
        const int64_t row = step * RPW + sub;
        const bool live = row < a.rows;
        const float mean = live ? a.mean[row] : 0.f, rstd = live ? a.rstd[row] : 0.f;
        float f[N * VEC], g[N * VEC], o[N * VEC];
        float c1 = 0.f, c2 = 0.f;
        // all three streams are asked for at once (fetching a row ahead instead took 10 % longer: fewer waves)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int e = (n * LPR + lane) * VEC;
            if (live && e < D) {
                re_load_some<T, VEC, ALIGNED>(static_cast<const T*>(a.s) + row * D + e, D - e, f + n * VEC);
                re_load_some<T, VEC, ALIGNED>(static_cast<const T*>(a.dy) + row * D + e, D - e, g + n * VEC);
                if (a.ds) re_load_some<T, VEC, ALIGNED>(static_cast<const T*>(a.ds) + row * D + e, D - e, o + n * VEC);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) f[n * VEC + v] = g[n * VEC + v] = 0.f;      // (dy 0: no part in any sum)
            }
        }
#pragma unroll
        for (int i = 0; i < N * VEC; ++i) {
            f[i] = (f[i] - mean) * rstd;
            dw[i] += g[i] * f[i];
            db[i] += g[i];
            g[i] *= w[i];
            c1 += g[i];
            c2 += g[i] * f[i];
        }
        row_sum2<LPR>(c1, c2, red);
        c1 *= inv_d;
        c2 *= inv_d;
        if (live) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int e = (n * LPR + lane) * VEC;
                if (e < D) {
#pragma unroll
                    for (int v = n * VEC; v < (n + 1) * VEC; ++v) {
                        const float d = rstd * (g[v] - c1 - f[v] * c2);
                        o[v] = a.ds ? o[v] + d : d;
                    }
                    re_store_some<T, VEC, ALIGNED>(static_cast<T*>(a.dx) + row * D + e, D - e, o + n * VEC);
                }
            }
        }
    }
    if (!a.part) return;
    float* part = a.part + (int64_t)blockIdx.x * 2 * D;
    // rows that share a workgroup: first the lanes of a wave that own the same columns, then the waves, in order
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float* acc = half ? db : dw;
        if constexpr (LPR < 64) {
#pragma unroll
            for (int i = 0; i < N * VEC; ++i) {
#pragma unroll
                for (int o = LPR; o < 64; o <<= 1) acc[i] += __shfl_xor(acc[i], o, 64);
            }
        }
        if constexpr (LPR < 256) {
            constexpr int PARTS = LPR < 64 ? 4 : RPW;
            const int at = LPR < 64 ? (int)(threadIdx.x >> 6) : sub;
            __syncthreads();
            if (LPR >= 64 || (threadIdx.x & 63) < LPR) {
#pragma unroll
                for (int i = 0; i < N * VEC; ++i) join[at * COLS + ((i / VEC) * LPR + lane) * VEC + i % VEC] = acc[i];
            }
            __syncthreads();
            for (int e = threadIdx.x; e < D; e += THREADS) {
                float t = 0.f;
#pragma unroll
                for (int p = 0; p < PARTS; ++p) t += join[p * COLS + e];
                part[half * D + e] = t;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N * VEC; ++i) {
                const int e = ((i / VEC) * LPR + lane) * VEC + i % VEC;
                if (e < D) part[half * D + e] = acc[i];
            }
        }
    }
}

// Rows too wide for the registers of a workgroup: the same two passes with the row read again from the caches.
template <class T>
__global__ __launch_bounds__(1024) void ln_fwd_wide_k(const ln_args a) {
    __shared__ float red[32];
    const int D = a.D;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + row * D;
        const T* r = a.r ? static_cast<const T*>(a.r) + row * D : nullptr;
        float sum = 0.f, sq = 0.f;
        for (int e = threadIdx.x; e < D; e += 1024) sum += (float)x[e] + (r ? (float)r[e] : 0.f);
        const float mean = row_sum<1024>(sum, red) / (float)D;
        for (int e = threadIdx.x; e < D; e += 1024) {
            const float d = (float)x[e] + (r ? (float)r[e] : 0.f) - mean;
            sq += d * d;
        }
        const float rstd = 1.f / sqrtf(row_sum<1024>(sq, red) / (float)D + a.eps);
        for (int e = threadIdx.x; e < D; e += 1024) {
            const float f = (float)x[e] + (r ? (float)r[e] : 0.f);
            const float w = a.w ? re_load_as_float(a.w, e, a.wtype) : 1.f, b = a.b ? re_load_as_float(a.b, e, a.wtype) : 0.f;
            static_cast<T*>(a.y)[row * D + e] = (T)((f - mean) * rstd * w + b);
            if (a.s) static_cast<T*>(a.s)[row * D + e] = (T)f;
        }
        if (threadIdx.x == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
    }
}
template <class T>
__global__ __launch_bounds__(1024) void ln_bwd_wide_k(const ln_bwd_args a) {
    __shared__ float red[32];
    const int D = a.D;
    float* part = a.part ? a.part + (int64_t)blockIdx.x * 2 * D : nullptr;
    bool first = true;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, first = false) {
        const T* s = static_cast<const T*>(a.s) + row * D;
        const T* dy = static_cast<const T*>(a.dy) + row * D;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float c1 = 0.f, c2 = 0.f;
        for (int e = threadIdx.x; e < D; e += 1024) {
            const float xhat = ((float)s[e] - mean) * rstd, d = (float)dy[e];
            const float g = d * (a.w ? re_load_as_float(a.w, e, a.wtype) : 1.f);
            c1 += g;
            c2 += g * xhat;
            if (part) {                       // (a column belongs to one thread in every row: its own partial)
                part[e] = (first ? 0.f : part[e]) + d * xhat;
                part[D + e] = (first ? 0.f : part[D + e]) + d;
            }
        }
        row_sum2<1024>(c1, c2, red);
        c1 /= (float)D;
        c2 /= (float)D;
        for (int e = threadIdx.x; e < D; e += 1024) {
            const float xhat = ((float)s[e] - mean) * rstd;
            const float g = (float)dy[e] * (a.w ? re_load_as_float(a.w, e, a.wtype) : 1.f);
            const float d = rstd * (g - c1 - xhat * c2);
            static_cast<T*>(a.dx)[row * D + e] = (T)(a.ds ? (float)static_cast<const T*>(a.ds)[row * D + e] + d : d);
        }
    }
}

// dw / db = the workgroups' partial rows added in order: 64 columns per workgroup, 16 waves with every 16th partial row each.
__global__ __launch_bounds__(1024) void ln_cols_k(const float* __restrict__ part, int groups, int D, void* dw, void* db, int32_t wtype) {
    __shared__ float t[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t col = (int64_t)blockIdx.x * 64 + lane;          // over [dw | db]
    float acc = 0.f;
    if (col < 2 * (int64_t)D) {
#pragma unroll 8
        for (int g = wave; g < groups; g += 16) acc += part[(int64_t)g * 2 * D + col];
    }
    t[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && col < 2 * (int64_t)D) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += t[i][lane];
        void* out = col < D ? dw : db;
        if (out) re_store_float(out, col < D ? col : col - D, wtype, s);
    }
}

// lanes per row and pieces per lane for a width: the narrowest form that holds the row
struct ln_form {
    int lpr, n;      // n = 0: ln_*_wide_k
};
ln_form ln_choose(int64_t D, int vec) {
    const int64_t p = (D + vec - 1) / vec;      // pieces
    if (p <= 16) return {16, 1};
    if (p <= 64) return {64, 1};
    if (p <= 128) return {64, 2};
    if (p <= 256) return {64, 4};
    if (p <= 512) return {256, 2};
    if (p <= 1024) return {256, 4};
    if (p <= 2048) return {1024, 2};
    return {1024, 0};
}

int ln_rows_per_wg(const ln_form f) { return f.lpr >= 256 ? 1 : 256 / f.lpr; }
// workgroups: at most `cap`, the rows spread evenly over them
unsigned ln_grid(int64_t rows, const ln_form f, int64_t cap) {
    const int64_t steps = re_cdiv(rows, ln_rows_per_wg(f));
    return (unsigned)re_cdiv(steps, re_cdiv(steps, cap));
}
// Workgroups at most.  More of them in flight do not read faster: 16384 x 4096 bf16, forward 122 us with 2048, 108 with 1024, 155 with 512; backward
// 119 with 512, 150 with 1024, 175 with 256.
constexpr int64_t LN_FWD_WGS = 1024, LN_BWD_WGS = 512;

#define LN_CASE(K, L, NN)                                                                                        \
    if (f.lpr == L && f.n == NN) {                                                                               \
        if (aligned) hipLaunchKernelGGL((K<T, L, V, NN, true>), dim3(grid), dim3(L > 256 ? L : 256), 0, st, a);  \
        else hipLaunchKernelGGL((K<T, L, V, NN, false>), dim3(grid), dim3(L > 256 ? L : 256), 0, st, a);         \
        return;                                                                                                  \
    }
#define LN_FORMS(K, KW)                                                                                          \
    constexpr int V = re_type<T>::VEC;                                                                           \
    LN_CASE(K, 16, 1) LN_CASE(K, 64, 1) LN_CASE(K, 64, 2) LN_CASE(K, 64, 4)                                      \
    LN_CASE(K, 256, 2) LN_CASE(K, 256, 4) LN_CASE(K, 1024, 2)                                                    \
    hipLaunchKernelGGL((KW<T>), dim3(grid), dim3(1024), 0, st, a);

template <class T>
void ln_fwd_launch(const ln_args& a, const ln_form f, bool aligned, unsigned grid, hipStream_t st) {
    LN_FORMS(ln_fwd_k, ln_fwd_wide_k)
}
template <class T>
void ln_bwd_launch(const ln_bwd_args& a, const ln_form f, bool aligned, unsigned grid, hipStream_t st) {
    LN_FORMS(ln_bwd_k, ln_bwd_wide_k)
}

bool ln_aligned(int64_t D, int32_t dtype, std::initializer_list<const void*> ps) {
    if (D % (16 / (int64_t)re_dtype_size(dtype))) return false;
    for (const void* p : ps)
        if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    return true;
}
ln_form ln_form_of(int64_t D, int32_t dtype) { return ln_choose(D, dtype == RE_F32 ? 4 : 8); }

}  // namespace

extern "C" int re_layer_norm_fwd(const void* x, const void* residual, const void* weight, const void* bias, int64_t rows, int64_t D,
                                 float eps, int32_t dtype, int32_t wtype, void* y, void* sum, float* mean, float* rstd,
                                 re_stream_t stream) {
    if (!re_dtype_size(dtype) || !re_dtype_size(wtype) || rows < 0 || D < 1) return RE_EINVAL;
    if (D > LN_MAX_D) return RE_EUNSUPPORTED;
    if (rows == 0) return RE_OK;
    if (!x || !y) return RE_EINVAL;
    re_clear_error();
    const ln_args a{x, residual, weight, bias, y, sum, mean, rstd, rows, (int32_t)D, wtype, eps};
    const bool aligned = ln_aligned(D, dtype, {x, residual, y, sum});
    const ln_form f = ln_form_of(D, dtype);
    const unsigned grid = ln_grid(rows, f, LN_FWD_WGS);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == RE_F32) ln_fwd_launch<float>(a, f, aligned, grid, st);
    else if (dtype == RE_BF16) ln_fwd_launch<re_bf16>(a, f, aligned, grid, st);
    else ln_fwd_launch<re_f16>(a, f, aligned, grid, st);
    return re_launch_status();
}

extern "C" size_t re_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t D) {
    if (rows < 1 || D < 1 || D > LN_MAX_D) return 0;
    return (size_t)(rows < LN_BWD_WGS ? rows : LN_BWD_WGS) * 2 * D * sizeof(float);
}

extern "C" int re_layer_norm_bwd(const void* dy, const void* s, const void* weight, const float* mean, const float* rstd,
                                 const void* dsum, int64_t rows, int64_t D, int32_t dtype, int32_t wtype, void* dx, void* dweight,
                                 void* dbias, void* ws, size_t ws_bytes, re_stream_t stream) {
    if (!re_dtype_size(dtype) || !re_dtype_size(wtype) || rows < 0 || D < 1) return RE_EINVAL;
    if (D > LN_MAX_D) return RE_EUNSUPPORTED;
    if (rows > 0 && (!dy || !s || !mean || !rstd || !dx)) return RE_EINVAL;
    const bool cols = dweight || dbias;
    if (cols && rows > 0 && (!ws || ws_bytes < re_layer_norm_bwd_workspace_bytes(rows, D))) return RE_EWORKSPACE;
    re_clear_error();
    hipStream_t st = (hipStream_t)stream;
    unsigned grid = 0;
    if (rows > 0) {
        const ln_bwd_args a{dy, s, weight, dsum, dx, mean, rstd, cols ? (float*)ws : nullptr, rows, (int32_t)D, wtype};
        const bool aligned = ln_aligned(D, dtype, {dy, s, dsum, dx});
        const ln_form f = ln_form_of(D, dtype);
        grid = ln_grid(rows, f, LN_BWD_WGS);
        if (dtype == RE_F32) ln_bwd_launch<float>(a, f, aligned, grid, st);
        else if (dtype == RE_BF16) ln_bwd_launch<re_bf16>(a, f, aligned, grid, st);
        else ln_bwd_launch<re_f16>(a, f, aligned, grid, st);
    }
    if (cols)
        hipLaunchKernelGGL(ln_cols_k, dim3((unsigned)re_cdiv(2 * D, 64)), dim3(1024), 0, st, (const float*)ws, (int)grid, (int)D, dweight,
                           dbias, wtype);
    return re_launch_status();
}
