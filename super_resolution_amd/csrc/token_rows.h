// The gated feed-forward block for few rows (up to 64): every weight is used once per row, so the time is that of reading the
// weights, and a tile of 128 rows would leave most of the chip idle.  A workgroup computes up to 16 output channels for all rows:
// its waves take the 128-byte blocks of k in turn, weights and rows straight from memory into the operands of the 16 x 16
// MFMA (weights as its rows, the tensor's rows as its columns, 16 at a time), and add up in the LDS in wave order.  A wave
// instruction reads 64 consecutive bytes of 16 rows.
// Measured (bf16): 1 row, 1024 x 4096: 5.0 + 5.1 us (16.8 and 8.4 MB of weights, the launch is half of it); 27 rows,
// 2048 x 8192: 17 us for the 67 MB of gate and up (3.9 TB/s; the tiles of 128 rows 21).  Its down product would take 20 us for
// 33 MB, since each of 256 workgroups also reads all 442 KB of rows from the L2 (4 channels a workgroup, which read the rows
// more often, 35; 16, which leave CUs idle, 22): with so many rows the split product takes it, in 15.
#pragma once
#include "token_gemm.h"

namespace sr355 {
namespace {

struct TokRowsArgs {
    const unsigned char *x, *w, *w2;      // rows; weights (GLU: gate and up) of one stride
    long long x_ld, w_ld;                 // bytes
    int rows, N, k_bytes;
    int channels;                         // output channels of a workgroup: 16, or fewer where that leaves CUs idle
    const void *bias, *bias2;
    void *out;                            // GLU: h
    const unsigned char *x_low;           // LOW: what h's rounding to the type left, added to the product
    void *out_low;                        // GLU: written where not null
    TokKept kept;                         // GLU: written where not null
    long long out_ld;                     // elements
    int n_store;                          // columns stored (GLU: up to the next eighth)
    int act;
};

template <typename T>
__device__ __forceinline__ void tok_mfma16(const tok_v4u &a, const tok_v4u &b, tok_f32x4 &c) {
    if constexpr (sizeof(T) == 4) {
        const tok_f32x4 fa = __builtin_bit_cast(tok_f32x4, a), fb = __builtin_bit_cast(tok_f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(fa[j], fb[j], c, 0, 0, 0);
    } else if constexpr (__is_same(T, bf16_t)) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(tok_bf16x8, a), __builtin_bit_cast(tok_bf16x8, b), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(tok_f16x8, a), __builtin_bit_cast(tok_f16x8, b), c, 0, 0, 0);
    }
}

// TG groups of 16 rows; GLU: two weights and the activation, else one weight.  LOW: the rows are the sum of two arrays, both
// multiplied with the weights as they pass: h keeps twice its bits in small blocks.
template <typename T, int TG, bool GLU, int WAVES, bool LOW>
__device__ __forceinline__ void tok_rows_body(const TokRowsArgs &p) {
    constexpr unsigned OUT = 0x80000000u;
    constexpr int Q = GLU ? 2 : 1, P = LOW ? 2 : 1;
    __shared__ float red[WAVES][Q * TG][16][17];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int i = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * p.channels;
    const __amdgpu_buffer_rsrc_t rw =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(p.w + n0 * p.w_ld), 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t rw2 =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>((GLU ? p.w2 : p.w) + n0 * p.w_ld), 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(p.x), 0, 0x7fffffff, 0x00020000);
    const __amdgpu_buffer_rsrc_t rl =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(LOW ? p.x_low : p.x), 0, 0x7fffffff, 0x00020000);
    const unsigned vw = i < p.channels && n0 + i < p.N ? (unsigned)(i * p.w_ld + g * 16) : OUT;
    unsigned vx[TG];
#pragma unroll
    for (int t = 0; t < TG; ++t) vx[t] = t * 16 + i < p.rows ? (unsigned)((t * 16 + i) * p.x_ld + g * 16) : OUT;
    tok_f32x4 acc[Q][TG];
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int t = 0; t < TG; ++t) acc[q][t] = tok_f32x4{0.f, 0.f, 0.f, 0.f};
    const int blocks = (p.k_bytes + 127) / 128;
    // Every workgroup reads the same rows.  Rows whose stride is a large power of two lie in one channel of the L2 at any k, so
    // the workgroups of an XCD (every eighth) start at different k, spread over all of it.
    const int first = (int)((long long)(blockIdx.x >> 3) % 32 * blocks / 32);
    // UN blocks' reads in flight (four take no less time); a block past the end reads zeros
    constexpr int UN = 2;
    for (int b = wave; b < blocks; b += WAVES * UN) {
        tok_v4u w[UN][Q][2], x[UN][P * TG][2];
#pragma unroll
        for (int k = 0; k < UN; ++k) {
            const int turn = b + k * WAVES, block = turn + first;
            const int at = turn < blocks ? (block < blocks ? block : block - blocks) * 128 : p.k_bytes;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                // (an offset beyond the buffer stays beyond it with the block's added, and what is read there is zero)
                const bool in = at + u * 64 + g * 16 < p.k_bytes;
                w[k][0][u] = __builtin_amdgcn_raw_buffer_load_b128(rw, in ? vw + at + u * 64 : OUT, 0, 0);
                if constexpr (GLU) w[k][Q - 1][u] = __builtin_amdgcn_raw_buffer_load_b128(rw2, in ? vw + at + u * 64 : OUT, 0, 0);
#pragma unroll
                for (int t = 0; t < TG; ++t) {
                    x[k][t][u] = __builtin_amdgcn_raw_buffer_load_b128(rx, in ? vx[t] + at + u * 64 : OUT, 0, 0);
                    if constexpr (LOW) x[k][TG + t][u] = __builtin_amdgcn_raw_buffer_load_b128(rl, in ? vx[t] + at + u * 64 : OUT, 0, 0);
                }
            }
        }
        __builtin_amdgcn_sched_barrier(0);                  // (all of them go out before the first is waited for)
#pragma unroll
        for (int k = 0; k < UN; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int t = 0; t < TG; ++t)
#pragma unroll
                    for (int q = 0; q < Q; ++q) {
                        tok_mfma16<T>(w[k][q][u], x[k][t][u], acc[q][t]);
                        if constexpr (LOW) tok_mfma16<T>(w[k][q][u], x[k][(P - 1) * TG + t][u], acc[q][t]);
                    }
    }
    // accumulator element e: n = 4 * (lane >> 4) + e, row = lane & 15
#pragma unroll
    for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int t = 0; t < TG; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[wave][q * TG + t][i][4 * g + e] = acc[q][t][e];
    __syncthreads();
    constexpr bool EXACT = sizeof(T) == 4;
    for (int k = threadIdx.x; k < 256 * TG; k += 64 * WAVES) {
        const int row = k >> 4, n = n0 + (k & 15);
        if (row >= p.rows || (k & 15) >= p.channels || n >= p.n_store) continue;
        float v[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            v[q] = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) v[q] += red[w][q * TG + (row >> 4)][row & 15][k & 15];
        }
        const long long at = row * p.out_ld + n;
        if (p.bias && n < p.N) v[0] += (float)((const T *)p.bias)[n];
        if constexpr (GLU) {
            if (p.bias2 && n < p.N) v[Q - 1] += (float)((const T *)p.bias2)[n];
            float a, d;
            if (p.act == SR355_ACT_SILU) tok_act_grad<EXACT, SR355_ACT_SILU>(v[0], a, d);
            else if (p.act == SR355_ACT_GELU) tok_act_grad<EXACT, SR355_ACT_GELU>(v[0], a, d);
            else if (p.act == SR355_ACT_RELU) tok_act_grad<EXACT, SR355_ACT_RELU>(v[0], a, d);
            else tok_act_grad<EXACT, SR355_ACT_SIGMOID>(v[0], a, d);
            // (hidden channels behind the last one: zeros, whatever an infinity in x makes of their zero weights)
            if (n >= p.N) a = d = v[Q - 1] = 0.f;
            const float h = a * v[Q - 1];
            const T high = (T)h;
            ((T *)p.out)[at] = high;
            if (p.out_low) ((T *)p.out_low)[at] = (T)(__builtin_isfinite((float)high) ? h - (float)high : 0.f);
            if (p.kept.a) {
                tok_keep<T>(p.kept.a, p.kept.a_low, at, a);
                tok_keep<T>(p.kept.d, p.kept.d_low, at, v[Q - 1] * d);
            }
        } else {
            ((T *)p.out)[at] = (T)v[0];
        }
    }
}

template <typename T, int TG, bool GLU, int WAVES, bool LOW>
__global__ __launch_bounds__(64 * WAVES) void tok_rows_kernel(TokRowsArgs p) {
    tok_rows_body<T, TG, GLU, WAVES, LOW>(p);
}

}  // namespace
}  // namespace sr355
