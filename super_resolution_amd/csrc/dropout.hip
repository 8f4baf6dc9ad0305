// Dropout with an optional skip: y = (keep ? x * scale : 0) + skip, and its gradient by the same kernel without a skip.
// The mask is never stored: element i of the tensor in row-major order takes 16 bits of Philox 4x32 (Salmon, Moraes, Dror
// and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011) with the key rng[0] and the counter (i / 8, rng[1], site),
// and is kept when they are at or over round(p * 65536); scale = 65536 / (65536 - round(p * 65536)), so the expectation is
// exact for the probability that is used.  Seven rounds: the paper's smallest number that passes all of its tests.
// Memory-bound: 2 or 3 elements moved per element against some 20 integer operations, which 16 bits an element (eight
// elements a call) keep below the memory's pace; 32 bits an element would be twice the work.  A thread owns a group of
// eight elements.  rng lives in device memory, so a captured graph's replays take the values it holds then.
#include "token_common.h"

namespace sr355 {

namespace {
struct DropArgs {
    const void *x, *skip;
    void *y;
    const long long *rng;
    long long n;
    unsigned threshold, site;
    float scale;
};

__device__ __forceinline__ void philox4x32_7(unsigned (&c)[4], unsigned k0, unsigned k1) {
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const unsigned long long a = (unsigned long long)c[0] * 0xD2511F53u, b = (unsigned long long)c[2] * 0xCD9E8D57u;
        const unsigned c1 = c[1], c3 = c[3];
        c[0] = (unsigned)(b >> 32) ^ c1 ^ k0, c[1] = (unsigned)b;
        c[2] = (unsigned)(a >> 32) ^ c3 ^ k1, c[3] = (unsigned)a;
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
}

// VEC: every pointer is 16-byte aligned, so a group of eight is one (16-bit types) or two (fp32) accesses.
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void dropout_kernel(DropArgs a) {
    constexpr int E = VEC ? 16 / sizeof(T) : 1;
    const unsigned long long seed = (unsigned long long)a.rng[0], step = (unsigned long long)a.rng[1];
    const long long groups = (a.n + 7) >> 3;
    for (long long g = (long long)blockIdx.x * 256 + threadIdx.x; g < groups; g += (long long)gridDim.x * 256) {
        unsigned c[4] = {(unsigned)g, (unsigned)(g >> 32), (unsigned)step, a.site};
        const T *x = (const T *)a.x + g * 8, *skip = (const T *)a.skip + g * 8;
        T *y = (T *)a.y + g * 8;
        const bool whole = g * 8 + 8 <= a.n;
        float v[8], s[8];
        if (VEC && whole) {
#pragma unroll
            for (int j = 0; j < 8; j += E) tok_load<T, E>(x + j, *reinterpret_cast<float(*)[E]>(v + j));
            if (a.skip) {
#pragma unroll
                for (int j = 0; j < 8; j += E) tok_load<T, E>(skip + j, *reinterpret_cast<float(*)[E]>(s + j));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                v[j] = g * 8 + j < a.n ? (float)x[j] : 0.f;
                s[j] = a.skip && g * 8 + j < a.n ? (float)skip[j] : 0.f;
            }
        }
        philox4x32_7(c, (unsigned)seed, (unsigned)(seed >> 32));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned bits = (c[j >> 1] >> (16 * (j & 1))) & 0xFFFFu;
            // (a dropped infinity or NaN is dropped: a choice, not a product with zero)
            v[j] = bits >= a.threshold ? v[j] * a.scale : 0.f;
            if (a.skip) v[j] += s[j];
        }
        if (VEC && whole) {
#pragma unroll
            for (int j = 0; j < 8; j += E) tok_store<T, E>(y + j, *reinterpret_cast<float(*)[E]>(v + j));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (g * 8 + j < a.n) y[j] = (T)v[j];
        }
    }
}

template <typename T>
int dropout_typed(const DropArgs &a, hipStream_t stream) {
    const long long groups = (a.n + 7) >> 3, wgs = tok_cdiv(groups, 256);
    const dim3 grid((unsigned)(wgs > (1 << 20) ? (1 << 20) : wgs));
    if (tok_aligned16(a.x) && tok_aligned16(a.skip) && tok_aligned16(a.y))
        hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(256), 0, stream, a);
    return check_hip(hipGetLastError(), "dropout launch");
}
}  // namespace

}  // namespace sr355

using namespace sr355;

extern "C" {

int sr355_dropout(const void *x, const void *skip, long long n, int dtype, double p, const long long *rng, unsigned site,
                  void *y, void *stream) {
    if (n < 1 || !tok_dtype_ok(dtype) || !(p >= 0.0 && p <= 1.0)) {
        set_error("dropout: bad arguments (n=%lld dtype=%d p=%g; at least one element, p in [0, 1])", n, dtype, p);
        return SR355_ERR_INVALID;
    }
    if (!x || !y || !rng) {
        set_error("dropout: null tensor");
        return SR355_ERR_INVALID;
    }
    DropArgs a = {};
    a.x = x, a.skip = skip, a.y = y, a.rng = rng, a.n = n, a.site = site;
    a.threshold = (unsigned)(p * 65536.0 + 0.5);
    a.scale = a.threshold < 65536u ? (float)(65536.0 / (65536.0 - a.threshold)) : 0.f;
    if (dtype == SR355_DTYPE_F32) return dropout_typed<float>(a, (hipStream_t)stream);
    if (dtype == SR355_DTYPE_BF16) return dropout_typed<bf16_t>(a, (hipStream_t)stream);
    return dropout_typed<f16_t>(a, (hipStream_t)stream);
}

}  // extern "C"
