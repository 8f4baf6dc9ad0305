// Layer normalisation over the channels of each row, forward and backward:
//     xh = (x - mean) * rstd, y = xh * w + b;   d = dy * w, dx = rstd * (d - mean(d) - xh * mean(d * xh)),
//     dw = sum over rows of dy * xh, db = sum over rows of dy.
// Both directions are bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.  A row is
// held in registers by L lanes (8 to 64 of a wave, or a workgroup of 256), so it is read once and the variance is the
// mean of squared deviations from the mean (E[x^2] - mean^2 loses it where the mean dominates).  The forward pass takes the
// channels' distances from the row's first one before it sums: what is common to them costs no bits, and equal channels are
// zeros (as sums of x, times the rounded 1 / C, 999 channels of 1000.1 gave a mean one step off and y = 0.04; it takes 1.4 us
// of 32768 x 1024 bf16's 26).  The backward pass takes the mean as it is stored, rounded to fp32.  Statistics, sums and the two
// row means are fp32.  The backward pass keeps dw / db of the lane's columns in registers over all rows of the workgroup and
// writes one partial row per workgroup; a second launch adds the partials in order.  No atomics.
#include <climits>

#include "token_common.h"

namespace sr355 {

namespace {
constexpr int LN_THREADS = 256;
constexpr int LN_MAX_PARTS = 512;      // two workgroups per CU
constexpr int LN_MOST = INT_MAX - 255; // channels: a thread's index steps by 256 behind the last one
constexpr int LN_LONG = 8192;          // channels from which on no type's row is held in registers (fp32 rows of whole units: 4096)

// Partial rows of dw and db, at most: rows beyond the registers have columns enough to fill the chip with fewer.
int ln_max_parts(int C) { return C <= LN_LONG ? LN_MAX_PARTS : C <= 65536 ? 64 : 8; }

// Sum over the lanes that hold one row.  L = 256: the four waves through LDS (red: 2 x 4 floats, alternating, so that
// one barrier per sum is enough).
template <int L>
__device__ __forceinline__ float row_sum(float v, float *red, int &turn) {
    if constexpr (L <= 64) return tok_lane_sum<L>(v);
    v = tok_lane_sum<64>(v);
    float *r = red + 8 * turn;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
    __syncthreads();
    return (r[0] + r[1]) + (r[2] + r[3]);
}
template <int L>
__device__ __forceinline__ void row_sum2(float &a, float &b, float *red, int &turn) {
    if constexpr (L <= 64) {
        a = tok_lane_sum<L>(a), b = tok_lane_sum<L>(b);
        return;
    }
    a = tok_lane_sum<64>(a), b = tok_lane_sum<64>(b);
    float *r = red + 8 * turn;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = a, r[4 + (threadIdx.x >> 6)] = b;
    __syncthreads();
    a = (r[0] + r[1]) + (r[2] + r[3]);
    b = (r[4] + r[5]) + (r[6] + r[7]);
}

struct LnArgs {
    const void *x, *dy, *w, *b;
    void *y;                    // forward: y; backward: dx (may be null)
    float *mean, *rstd;         // forward: written; backward: read
    float *parts;               // backward: [gridDim.x][2][C]
    long long rows, x_ld, dy_ld;
    int C, w32;
    float eps;
};

// What a row's channels are measured from: its first one, unless that is so large that a difference could overflow (or no number).
__device__ __forceinline__ float ln_origin(float first) { return fabsf(first) < 0x1p100f ? first : 0.f; }

// The row in registers: lane l of L holds units l, l + L, ... of E elements.
template <typename T, int E, int L, int U>
__global__ __launch_bounds__(LN_THREADS) void ln_fwd_kernel(LnArgs a) {
    constexpr int ROWS = LN_THREADS / L;
    __shared__ float red[16];
    int turn = 0;
    const int l = threadIdx.x % L;
    const float inv_c = 1.0f / (float)a.C;
    for (long long row = (long long)blockIdx.x * ROWS + threadIdx.x / L; row < a.rows; row += (long long)gridDim.x * ROWS) {
        const T *x = (const T *)a.x + row * a.x_ld;
        float v[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = (u * L + l) * E;
#pragma unroll
            for (int j = 0; j < E; ++j) v[u][j] = 0.f;
            if (c < a.C) tok_load<T, E>(x + c, v[u]);
        }
        float first;                                        // (the row's first lane has its first channel)
        if constexpr (L < 64) first = __shfl(v[0][0], 0, L);
        else if constexpr (L == 64) first = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v[0][0])));
        else first = (float)x[0];
        const float origin = ln_origin(first);
        float s = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if ((u * L + l) * E >= a.C) continue;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[u][j] -= origin;
                s += v[u][j];
            }
        }
        const float mean = row_sum<L>(s, red, turn) * inv_c;
        if (l == 0 && a.mean) a.mean[row] = origin + mean;
        float q = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const bool in = (u * L + l) * E < a.C;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[u][j] -= mean;
                if (in) q += v[u][j] * v[u][j];
            }
        }
        const float rstd = 1.0f / sqrtf(row_sum<L>(q, red, turn) * inv_c + a.eps);
        if (l == 0 && a.mean) a.rstd[row] = rstd;
        T *y = (T *)a.y + row * (long long)a.C;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = (u * L + l) * E;
            if (c >= a.C) continue;
            float w[E], b[E];
            if (a.w) tok_load_param<T, E>(a.w, a.w32, c, w);
            if (a.b) tok_load_param<T, E>(a.b, a.w32, c, b);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                float o = v[u][j] * rstd;
                if (a.w) o *= w[j];
                if (a.b) o += b[j];
                v[u][j] = o;
            }
            tok_store<T, E>(y + c, v[u]);
        }
    }
}

template <typename T, int E, int L, int U>
__global__ __launch_bounds__(LN_THREADS) void ln_bwd_kernel(LnArgs a) {
    constexpr int ROWS = LN_THREADS / L;
    __shared__ float red[16];
    __shared__ float comb[L == LN_THREADS ? 1 : LN_THREADS * E];
    int turn = 0;
    const int l = threadIdx.x % L;
    const float inv_c = 1.0f / (float)a.C;
    float w[U][E], sw[U][E], sb[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int c = (u * L + l) * E;
#pragma unroll
        for (int j = 0; j < E; ++j) w[u][j] = 1.f, sw[u][j] = sb[u][j] = 0.f;
        if (a.w && c < a.C) tok_load_param<T, E>(a.w, a.w32, c, w[u]);
    }
    for (long long row = (long long)blockIdx.x * ROWS + threadIdx.x / L; row < a.rows; row += (long long)gridDim.x * ROWS) {
        const T *x = (const T *)a.x + row * a.x_ld, *dy = (const T *)a.dy + row * a.dy_ld;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float xh[U][E], d[U][E];
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = (u * L + l) * E;
#pragma unroll
            for (int j = 0; j < E; ++j) xh[u][j] = mean, d[u][j] = 0.f;
            if (c < a.C) {
                tok_load<T, E>(x + c, xh[u]);
                tok_load<T, E>(dy + c, d[u]);
            }
#pragma unroll
            for (int j = 0; j < E; ++j) {
                xh[u][j] = (xh[u][j] - mean) * rstd;
                sw[u][j] += d[u][j] * xh[u][j];
                sb[u][j] += d[u][j];
                d[u][j] *= w[u][j];
                s += d[u][j];
                q += d[u][j] * xh[u][j];
            }
        }
        if (!a.y) continue;
        row_sum2<L>(s, q, red, turn);
        s *= inv_c, q *= inv_c;
        T *dx = (T *)a.y + row * (long long)a.C;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = (u * L + l) * E;
            if (c >= a.C) continue;
#pragma unroll
            for (int j = 0; j < E; ++j) d[u][j] = rstd * (d[u][j] - s - xh[u][j] * q);
            tok_store<T, E>(dx + c, d[u]);
        }
    }
    if (!a.parts) return;
    // the row groups of the workgroup in order, then one partial row per workgroup
    float *part = a.parts + (size_t)blockIdx.x * 2 * a.C;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = (u * L + l) * E;
            float t[E];
#pragma unroll
            for (int j = 0; j < E; ++j) t[j] = which ? sb[u][j] : sw[u][j];
            if constexpr (ROWS > 1) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < E; ++j) comb[j * LN_THREADS + threadIdx.x] = t[j];
                __syncthreads();
                if (threadIdx.x < L) {
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        t[j] = 0.f;
                        for (int r = 0; r < ROWS; ++r) t[j] += comb[j * LN_THREADS + r * L + threadIdx.x];
                    }
                }
            }
            if (threadIdx.x < L && c < a.C) {
#pragma unroll
                for (int j = 0; j < E; ++j) part[(size_t)which * a.C + c + j] = t[j];
            }
        }
    }
}

// Rows too long for the registers of a workgroup: a workgroup per row that reads it three times (forward) or twice
// (backward), from L2 after the first time.
template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_fwd_long_kernel(LnArgs a) {
    __shared__ float red[16];
    int turn = 0;
    const float inv_c = 1.0f / (float)a.C;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_ld;
        const float origin = ln_origin((float)x[0]);
        float s = 0.f, q = 0.f;
        for (int c = threadIdx.x; c < a.C; c += LN_THREADS) s += (float)x[c] - origin;
        const float mean = row_sum<LN_THREADS>(s, red, turn) * inv_c;
        for (int c = threadIdx.x; c < a.C; c += LN_THREADS) {
            const float d = ((float)x[c] - origin) - mean;
            q += d * d;
        }
        const float rstd = 1.0f / sqrtf(row_sum<LN_THREADS>(q, red, turn) * inv_c + a.eps);
        if (threadIdx.x == 0 && a.mean) a.mean[row] = origin + mean, a.rstd[row] = rstd;
        T *y = (T *)a.y + row * (long long)a.C;
        for (int c = threadIdx.x; c < a.C; c += LN_THREADS) {
            float w[1] = {1.f}, b[1] = {0.f};
            if (a.w) tok_load_param<T, 1>(a.w, a.w32, c, w);
            if (a.b) tok_load_param<T, 1>(a.b, a.w32, c, b);
            y[c] = (T)((((float)x[c] - origin) - mean) * rstd * w[0] + b[0]);
        }
    }
}

template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_bwd_long_kernel(LnArgs a) {
    __shared__ float red[16];
    int turn = 0;
    const float inv_c = 1.0f / (float)a.C;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_ld, *dy = (const T *)a.dy + row * a.dy_ld;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s = 0.f, q = 0.f;
        for (int c = threadIdx.x; c < a.C; c += LN_THREADS) {
            float w[1] = {1.f};
            if (a.w) tok_load_param<T, 1>(a.w, a.w32, c, w);
            const float d = (float)dy[c] * w[0];
            s += d;
            q += d * ((float)x[c] - mean) * rstd;
        }
        row_sum2<LN_THREADS>(s, q, red, turn);
        s *= inv_c, q *= inv_c;
        T *dx = (T *)a.y + row * (long long)a.C;
        for (int c = threadIdx.x; c < a.C; c += LN_THREADS) {
            float w[1] = {1.f};
            if (a.w) tok_load_param<T, 1>(a.w, a.w32, c, w);
            dx[c] = (T)(rstd * ((float)dy[c] * w[0] - s - ((float)x[c] - mean) * rstd * q));
        }
    }
}

// dw / db of long rows: workgroup (block of 256 columns, part), one column per thread.
template <typename T>
__global__ __launch_bounds__(LN_THREADS) void ln_columns_long_kernel(LnArgs a) {
    const int c = blockIdx.x * LN_THREADS + threadIdx.x;
    if (c >= a.C) return;
    float sw = 0.f, sb = 0.f;
    for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float d = (float)((const T *)a.dy)[row * a.dy_ld + c];
        sw += d * (((float)((const T *)a.x)[row * a.x_ld + c] - a.mean[row]) * a.rstd[row]);
        sb += d;
    }
    float *part = a.parts + (size_t)blockIdx.y * 2 * a.C;
    part[c] = sw;
    part[(size_t)a.C + c] = sb;
}

// out[k][j] = sum over parts p, in order, of parts[p * stride + first[k] + j]: the tail of every two-level column sum.
// A workgroup adds 64 columns, sixteen waves taking a sixteenth of the parts each (four waves: 7.7 us for 512 parts).
struct SumArgs {
    const float *parts;
    long long stride, first[4];
    void *out[4];
    int count[4];
    int n_parts, out_dtype;
};
constexpr int SUM_WAVES = 16;
constexpr int SUM_WGS = 1 << 21;       // a grid axis holds fewer than 2^32 threads (more are dropped without an error)
__global__ __launch_bounds__(64 * SUM_WAVES) void tok_sum_parts_kernel(SumArgs a) {
    __shared__ float red[SUM_WAVES][64];
    const int k = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (long long first = blockIdx.x * 64LL; first < a.count[k]; first += gridDim.x * 64LL) {
        const long long j = first + lane;
        float s = 0.f;
        if (j < a.count[k]) {
            const float *p = a.parts + a.first[k] + j;
            const int lo = (int)((long long)a.n_parts * wave / SUM_WAVES), hi = (int)((long long)a.n_parts * (wave + 1) / SUM_WAVES);
#pragma unroll 8
            for (int i = lo; i < hi; ++i) s += p[(size_t)i * a.stride];
        }
        __syncthreads();                                    // (the columns before these have been added)
        red[wave][lane] = s;
        __syncthreads();
        if (wave || j >= a.count[k]) continue;
        s = 0.f;
#pragma unroll
        for (int w = 0; w < SUM_WAVES; ++w) s += red[w][lane];
        if (a.out_dtype == SR355_DTYPE_F32) ((float *)a.out[k])[j] = s;
        else if (a.out_dtype == SR355_DTYPE_BF16) ((bf16_t *)a.out[k])[j] = (bf16_t)s;
        else ((f16_t *)a.out[k])[j] = (f16_t)s;
    }
}

int ln_grid(long long rows, int rows_per_wg, int most) {
    const long long n = tok_cdiv(rows, rows_per_wg);
    return (int)(n < 1 ? 1 : (n > most ? most : n));
}

// The smallest variant that holds C channels: (elements per access, lanes per row, units per lane).  16-byte accesses
// need the channel count, the row strides and the pointers to be multiples of 16 bytes; other rows go element by element.
template <typename T, typename F>
int ln_dispatch(bool vec, int C, F &&f) {
    constexpr int E = 16 / sizeof(T);
    if (vec) {
        if (C <= 8 * E) return f.template run<T, E, 8, 1>();
        if (C <= 16 * E) return f.template run<T, E, 16, 1>();
        if (C <= 32 * E) return f.template run<T, E, 32, 1>();
        if (C <= 64 * E) return f.template run<T, E, 64, 1>();
        if (C <= 128 * E) return f.template run<T, E, 64, 2>();
        if (C <= 256 * E) return f.template run<T, E, 64, 4>();
        if (C <= 512 * E) return f.template run<T, E, 256, 2>();
        if (C <= 1024 * E) return f.template run<T, E, 256, 4>();
    } else {
        if (C <= 64) return f.template run<T, 1, 16, 4>();
        if (C <= 256) return f.template run<T, 1, 64, 4>();
        if (C <= 1024) return f.template run<T, 1, 64, 16>();
        if (C <= 4096) return f.template run<T, 1, 256, 16>();
        if (C <= 8192) return f.template run<T, 1, 256, 32>();
    }
    return f.template run_long<T>();
}

struct LnForward {
    LnArgs a;
    hipStream_t stream;
    template <typename T, int E, int L, int U>
    int run() {
        hipLaunchKernelGGL((ln_fwd_kernel<T, E, L, U>), dim3(ln_grid(a.rows, LN_THREADS / L, 1 << 20)), dim3(LN_THREADS), 0,
                           stream, a);
        return check_hip(hipGetLastError(), "layer_norm_fwd launch");
    }
    template <typename T>
    int run_long() {
        hipLaunchKernelGGL((ln_fwd_long_kernel<T>), dim3(ln_grid(a.rows, 1, 1 << 20)), dim3(LN_THREADS), 0, stream, a);
        return check_hip(hipGetLastError(), "layer_norm_fwd launch");
    }
};

struct LnBackward {
    LnArgs a;
    hipStream_t stream;
    int *n_parts;
    template <typename T, int E, int L, int U>
    int run() {
        *n_parts = ln_grid(a.rows, LN_THREADS / L, LN_MAX_PARTS);
        hipLaunchKernelGGL((ln_bwd_kernel<T, E, L, U>), dim3(*n_parts), dim3(LN_THREADS), 0, stream, a);
        return check_hip(hipGetLastError(), "layer_norm_bwd launch");
    }
    template <typename T>
    int run_long() {
        if (a.y) hipLaunchKernelGGL((ln_bwd_long_kernel<T>), dim3(ln_grid(a.rows, 1, 1 << 20)), dim3(LN_THREADS), 0, stream, a);
        *n_parts = ln_grid(a.rows, 64, ln_max_parts(a.C) < 64 ? ln_max_parts(a.C) : 64);
        if (a.parts)
            hipLaunchKernelGGL((ln_columns_long_kernel<T>), dim3((unsigned)tok_cdiv(a.C, LN_THREADS), *n_parts), dim3(LN_THREADS), 0,
                               stream, a);
        return check_hip(hipGetLastError(), "layer_norm_bwd launch");
    }
};

template <typename F>
int ln_by_type(int dtype, bool vec, int C, F &f) {
    if (dtype == SR355_DTYPE_F32) return ln_dispatch<float>(vec, C, f);
    if (dtype == SR355_DTYPE_BF16) return ln_dispatch<bf16_t>(vec, C, f);
    return ln_dispatch<f16_t>(vec, C, f);
}

bool ln_vec(int dtype, int C, long long ld0, long long ld1, const void *p0, const void *p1, const void *p2) {
    const int e = dtype == SR355_DTYPE_F32 ? 4 : 8;
    return C % e == 0 && ld0 % e == 0 && ld1 % e == 0 && tok_aligned16(p0) && tok_aligned16(p1) && tok_aligned16(p2);
}

bool ln_args_ok(const char *who, long long rows, int C, int dtype, long long ld0, long long ld1, const void *w, int w_dtype) {
    if (rows < 0 || C < 1 || C > LN_MOST || !tok_dtype_ok(dtype) || ld0 < C || ld1 < C ||
        (w && w_dtype != dtype && w_dtype != SR355_DTYPE_F32)) {
        set_error("%s: bad arguments (rows=%lld, C=%d channels of at most 2^31 - 256, dtype=%d, row strides %lld and %lld elements, parameters of type %d: the "
                  "activations' type or fp32)", who, rows, C, dtype, ld0, ld1, w_dtype);
        return false;
    }
    return true;
}
}  // namespace

int launch_tok_sum_parts(const float *parts, int n_parts, long long stride, const long long *first, const int *count, void *const *out,
                         int n_out, int out_dtype, hipStream_t stream) {
    SumArgs s = {};
    s.parts = parts, s.stride = stride, s.n_parts = n_parts, s.out_dtype = out_dtype;
    int n = 0, most = 0;
    for (int k = 0; k < n_out; ++k) {
        if (!out[k]) continue;
        s.first[n] = first[k], s.count[n] = count[k], s.out[n] = out[k];
        if (count[k] > most) most = count[k];
        ++n;
    }
    if (n == 0 || most == 0) return SR355_OK;
    const long long wgs = tok_cdiv(most, 64);
    hipLaunchKernelGGL(tok_sum_parts_kernel, dim3((unsigned)(wgs < SUM_WGS ? wgs : SUM_WGS), n), dim3(64 * SUM_WAVES), 0, stream, s);
    return check_hip(hipGetLastError(), "column sum launch");
}

}  // namespace sr355

using namespace sr355;

extern "C" {

int sr355_layer_norm_fwd(const void *x, long long rows, int C, long long x_ld, int dtype, const void *w, const void *b,
                         int w_dtype, float eps, void *y, float *mean, float *rstd, void *stream) {
    if (!ln_args_ok("layer_norm_fwd", rows, C, dtype, x_ld, C, w ? w : b, w_dtype)) return SR355_ERR_INVALID;
    if (rows == 0) return SR355_OK;
    if (!x || !y || (mean == nullptr) != (rstd == nullptr) || !(eps >= 0.f)) {
        set_error("layer_norm_fwd: null tensor, only one of mean / rstd, or a negative eps");
        return SR355_ERR_INVALID;
    }
    LnForward f = {};
    f.a.x = x, f.a.w = w, f.a.b = b, f.a.y = y, f.a.mean = mean, f.a.rstd = rstd;
    f.a.rows = rows, f.a.x_ld = x_ld, f.a.C = C, f.a.w32 = w_dtype == SR355_DTYPE_F32, f.a.eps = eps;
    f.stream = (hipStream_t)stream;
    return ln_by_type(dtype, ln_vec(dtype, C, x_ld, C, x, y, y), C, f);
}

size_t sr355_layer_norm_bwd_workspace_bytes(int C) {
    if (C < 1 || C > LN_MOST) {
        set_error("layer_norm_bwd_workspace_bytes: C=%d channels", C);
        return 0;
    }
    return (size_t)ln_max_parts(C) * 2 * C * sizeof(float);
}

int sr355_layer_norm_bwd(const void *dy, long long dy_ld, const void *x, long long x_ld, long long rows, int C, int dtype,
                         const void *w, int w_dtype, const float *mean, const float *rstd, void *dx, void *dw, void *db,
                         void *workspace, size_t workspace_bytes, void *stream) {
    if (!ln_args_ok("layer_norm_bwd", rows, C, dtype, x_ld, dy_ld, w, w_dtype)) return SR355_ERR_INVALID;
    if ((dw || db) && w_dtype != dtype && w_dtype != SR355_DTYPE_F32) {
        set_error("layer_norm_bwd: parameter gradients of the activations' type or fp32 (got type %d)", w_dtype);
        return SR355_ERR_INVALID;
    }
    if ((rows > 0 && (!dy || !x || !mean || !rstd)) ||
        ((dw || db) && (!workspace || !tok_aligned16(workspace) || workspace_bytes < sr355_layer_norm_bwd_workspace_bytes(C)))) {
        set_error("layer_norm_bwd: null tensor, or a workspace that is not 16-byte aligned or smaller than %zu bytes",
                  sr355_layer_norm_bwd_workspace_bytes(C));
        return SR355_ERR_INVALID;
    }
    if (!dx && !dw && !db) return SR355_OK;
    if (rows == 0 && !dw && !db) return SR355_OK;
    int n_parts = 0;
    if (rows > 0) {
        LnBackward f = {};
        f.a.x = x, f.a.dy = dy, f.a.w = w, f.a.y = dx;
        f.a.mean = const_cast<float *>(mean), f.a.rstd = const_cast<float *>(rstd);
        f.a.parts = (dw || db) ? (float *)workspace : nullptr;
        f.a.rows = rows, f.a.x_ld = x_ld, f.a.dy_ld = dy_ld, f.a.C = C, f.a.w32 = w_dtype == SR355_DTYPE_F32;
        f.stream = (hipStream_t)stream, f.n_parts = &n_parts;
        const int rc = ln_by_type(dtype, ln_vec(dtype, C, x_ld, dy_ld, x, dy, dx), C, f);
        if (rc != SR355_OK || !f.a.parts) return rc;
    }
    const long long first[2] = {0, C};
    const int count[2] = {C, C};
    void *const out[2] = {dw, db};
    return launch_tok_sum_parts((const float *)workspace, n_parts, 2LL * C, first, count, out, 2, w_dtype, (hipStream_t)stream);
}

}  // extern "C"
