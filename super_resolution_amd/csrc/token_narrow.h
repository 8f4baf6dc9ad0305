// The gated feed-forward block of narrow rows (up to 128 channels, 16-bit types, nothing kept) in one launch: the hidden
// channels never leave the registers.  Through memory they would be most of the traffic: 262144 x 64 x 256 reads and writes
// 67 MB of rows, and 268 MB of hidden channels.
// A wave owns 32 rows: their x as MFMA operands (read once) and their y as accumulators.  The workgroup's four waves walk
// the hidden channels in chunks of HC; the chunk's rows of the gate and up weights and columns of the down weight are copied
// into the LDS (two buffers, one barrier a chunk).  Per 32 hidden channels: g and u by MFMA, the activation on the
// accumulators, and h as the next product's operand straight from there: a lane of the accumulator holds, of each 16 hidden
// channels, rows 0-3 and 8-11 or 4-7 and 12-15 of the weight's image, and an operand wants eight consecutive k, so the
// weight rows are placed with their second and third quads exchanged.
// Bound by the vector units: the activation is some 20 instructions per element and lane against 12 MFMAs per 16 elements.
// Measured (bf16, 262144 x 64 x 256): gelu with biases 67 us, without 59, silu 41, relu 35; the two launches through memory
// take 156 us for the first.  64 rows a wave spill registers (113 us); the activation as a branch inside the loop 75 us.
#pragma once
#include "token_gemm.h"

namespace sr355 {
namespace {

struct TokNarrowArgs {
    const unsigned char *x, *wg, *wu, *wd;
    const unsigned char *bg, *bu;         // padded to units, or null
    const void *bd;
    void *y;
    long long rows, x_ld, w_ld, wd_ld;    // bytes
    long long y_ld;                       // elements
    int C, F, act;
};

template <int ROW_UNITS>
__device__ __forceinline__ int tok_spread(int r) {   // permutation of a row's units, as in TokImage::rot
    return ROW_UNITS == 16 ? r & 15 : ROW_UNITS == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
}

template <int OFF>
__device__ __forceinline__ void tok_read_unit(tok_v4u &f, unsigned addr) {
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=&v"(f) : "v"(addr), "n"(OFF) : "memory");
}

template <int CP>
struct TokNarrow {
    static constexpr int HC = 4096 / CP;                     // hidden channels of a chunk: its three parts are 8 KB each
    static constexpr int PART = 8192, STAGE = 3 * PART + 1024;   // and the chunk's biases
    static constexpr int ROWS = 128;                         // of a workgroup
};

template <typename T, int CP, int KIND, bool BIAS>
__device__ __forceinline__ void tok_narrow_body(const TokNarrowArgs &p) {
    typedef TokNarrow<CP> N;
    constexpr int HC = N::HC, RB = CP * 2, HB = HC * 2;      // bytes of a row of the gate / up and of the down image
    constexpr int UR = RB / 16, UH = HB / 16;
    constexpr int KS = CP / 16, SUBS = HC / 32, CB = CP / 32;
    constexpr unsigned OUT = 0x80000000u;
    __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * N::STAGE];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l = lane & 31, half = lane >> 5;
    const long long row0 = (long long)blockIdx.x * N::ROWS + wave * 32;

    // x: operand of row l, k = 16 s + 8 half ..
    tok_v4u x[KS];
    {
        const __amdgpu_buffer_rsrc_t r =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(p.x + row0 * p.x_ld), 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int s = 0; s < KS; ++s)
            x[s] = __builtin_amdgcn_raw_buffer_load_b128(
                r, row0 + l < p.rows && 16 * s + 8 * half < p.C ? (int)(l * p.x_ld + (2 * s + half) * 16) : (int)OUT, 0, 0);
    }
    // sources of this wave's six copies, relative to the chunk's corner: two of each part
    unsigned v[6];
    short hid[6];                                            // hidden channel of the line / unit inside the chunk
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        const int at = ((i & 1) * 4 + wave) * 64 + lane;     // unit of the part's image
        if (i < 4) {
            const int line = at / UR, unit = (at % UR) ^ tok_spread<UR>(line);
            const int h = (line & ~12) | ((line & 4) << 1) | ((line & 8) >> 1);
            v[i] = unit * 8 < p.C ? (unsigned)(h * p.w_ld + unit * 16) : OUT;
            hid[i] = h;
        } else {
            const int line = at / UH, unit = (at % UH) ^ tok_spread<UH>(line);
            v[i] = line < p.C ? (unsigned)(line * p.wd_ld + unit * 16) : OUT;
            hid[i] = unit * 8;
        }
    }
    auto copy = [&](int chunk, int slot) {
        const int left = p.F - chunk * HC;
        unsigned char *const dst = smem + slot * N::STAGE;
        const unsigned char *const base[3] = {p.wg + (long long)chunk * HC * p.w_ld, p.wu + (long long)chunk * HC * p.w_ld,
                                              p.wd + (long long)chunk * HB};
#pragma unroll
        for (int i = 0; i < 6; ++i) {
            const __amdgpu_buffer_rsrc_t r =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(base[i >> 1]), 0, 0x7fffffff, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (tok_lds_void *)(dst + (i >> 1) * N::PART + ((i & 1) * 4 + wave) * 1024), 16,
                                                     hid[i] < left ? v[i] : OUT, 0, 0, 0);
        }
        if (BIAS && wave < 2) {
            // wave 0 the gate biases, wave 1 the up biases, zeros where there are none
            const unsigned char *b = wave ? p.bu : p.bg;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<unsigned char *>(b ? b + (long long)chunk * HB : p.wg), 0, b ? 0x7fffffff : 0, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (tok_lds_void *)(dst + 3 * N::PART + wave * 512), 4,
                                                     lane < HB / 4 && (lane >> 2) * 8 < left ? lane * 4 : OUT, 0, 0, 0);
        }
    };

    const unsigned lds0 = (unsigned)(size_t)(tok_lds_void *)smem;
    unsigned ow[KS], od[SUBS * 2];
#pragma unroll
    for (int s = 0; s < KS; ++s) ow[s] = l * RB + ((2 * s + half) ^ tok_spread<UR>(l)) * 16;
#pragma unroll
    for (int s = 0; s < SUBS * 2; ++s) od[s] = 2 * N::PART + l * HB + ((2 * s + half) ^ tok_spread<UH>(l)) * 16;

    tok_f32x16 y[CB];
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) y[c][e] = 0.f;

    // `left`: hidden channels from the chunk's first one on
    auto chunk_product = [&](unsigned base, int left) {
        tok_static_for<SUBS>([&](auto sub) {
            constexpr int SUB = decltype(sub)::value;
            tok_v4u fg[KS], fu[KS], fd[CB][2], bias[4];
            tok_static_for<KS>([&](auto s) {
                constexpr int S = decltype(s)::value;
                tok_read_unit<SUB * 32 * RB>(fg[S], base + ow[S]);
                tok_read_unit<N::PART + SUB * 32 * RB>(fu[S], base + ow[S]);
            });
            // biases of hidden channels 8 half .. and 16 + 8 half .. of the 32
            if constexpr (BIAS) tok_static_for<2>([&](auto q) {
                constexpr int Q = decltype(q)::value;
                tok_read_unit<3 * N::PART + SUB * 64 + Q * 32>(bias[Q], base + half * 16);
                tok_read_unit<3 * N::PART + 512 + SUB * 64 + Q * 32>(bias[2 + Q], base + half * 16);
            });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(fg[s]), "+v"(fu[s]));
            if constexpr (BIAS) asm volatile("" : "+v"(bias[0]), "+v"(bias[1]), "+v"(bias[2]), "+v"(bias[3]));
            tok_f32x16 g, u;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                g[e] = u[e] = 0.f;
                if constexpr (BIAS) {
                    T b[2];
                    const unsigned wg = bias[e >> 3][(e & 7) >> 1], wu = bias[2 + (e >> 3)][(e & 7) >> 1];
                    __builtin_memcpy(b, &wg, 4);
                    g[e] = (float)b[e & 1];
                    __builtin_memcpy(b, &wu, 4);
                    u[e] = (float)b[e & 1];
                }
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                tok_mfma<T>(fg[s], x[s], g);
                tok_mfma<T>(fu[s], x[s], u);
            }
            tok_static_for<CB>([&](auto c) {
                constexpr int C = decltype(c)::value;
                tok_read_unit<C * 32 * HB>(fd[C][0], base + od[SUB * 2]);
                tok_read_unit<C * 32 * HB>(fd[C][1], base + od[SUB * 2 + 1]);
            });
            T h[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) h[e] = (T)(tok_act<false, KIND>(g[e]) * u[e]);
            tok_v4u fh[2];
            __builtin_memcpy(fh, h, 32);
            // hidden channels behind the last one are zeros, whatever an infinity in x makes of their zero weights; element e is
            // channel (e & 7) + 8 half + 16 (e >> 3) of the 32
            if (left < (SUB + 1) * 32) {
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const int behind = SUB * 32 + (e & 7) + 8 * half + 16 * (e >> 3) - left;
                    fh[e >> 3][(e & 7) >> 1] &= behind >= 0 ? 0u : behind == -1 ? 0x0000ffffu : 0xffffffffu;
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int c = 0; c < CB; ++c) {
                asm volatile("" : "+v"(fd[c][0]), "+v"(fd[c][1]));
                tok_mfma<T>(fd[c][0], fh[0], y[c]);
                tok_mfma<T>(fd[c][1], fh[1], y[c]);
            }
        });
    };
    const int chunks = (p.F + HC - 1) / HC;
    copy(0, 0);
    for (int c = 0; c < chunks; ++c) {
        // this chunk has landed and nobody reads the other buffer any more
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (c + 1 < chunks) copy(c + 1, (c + 1) & 1);
        const unsigned base = lds0 + (c & 1) * N::STAGE;
        chunk_product(base, p.F - c * HC);
    }
    __builtin_amdgcn_s_barrier();                            // the last chunk's copies have all landed (waited for above)
    asm volatile("" ::: "memory");
    // y: lane (row l, channels 32 c + 8 q + 4 half ..) -> rows of 16-byte units
    unsigned char *const turn = smem + wave * 32 * RB;
    const int unit = lane % UR, col = unit * 8;
    const bool wide = (p.C & 7) == 0 && (p.y_ld & 7) == 0 && ((size_t)p.y & 15) == 0;
    constexpr int RPI = 64 / UR;
#pragma unroll
    for (int c = 0; c < CB; ++c)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int at = 32 * c + 8 * q + 4 * half;
            T o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float b = 0.f;
                if (p.bd && at + j < p.C) b = (float)((const T *)p.bd)[at + j];
                o[j] = (T)(y[c][4 * q + j] + b);
            }
            tok_v2u raw;
            __builtin_memcpy(&raw, o, 8);
            *reinterpret_cast<tok_v2u *>(turn + l * RB + ((at / 8) ^ tok_spread<UR>(l)) * 16 + (at % 8) * 2) = raw;
        }
    asm volatile("" ::: "memory");                           // (the lanes of a wave read what others of them wrote, in order)
    for (int r = lane / UR; r < 32; r += RPI) {
        const long long m = row0 + r;
        if (m >= p.rows || col >= p.C) continue;
        const tok_v4u o = *reinterpret_cast<const tok_v4u *>(turn + r * RB + (unit ^ tok_spread<UR>(r)) * 16);
        T *dst = (T *)p.y + m * p.y_ld + col;
        if (wide) {
            *reinterpret_cast<tok_v4u *>(dst) = o;
        } else {
            T t[8];
            __builtin_memcpy(t, &o, 16);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (col + j < p.C) dst[j] = t[j];
        }
    }
}

template <typename T, int CP, int KIND, bool BIAS>
__global__ __launch_bounds__(256, 2) void tok_narrow_kernel(TokNarrowArgs p) {
    tok_narrow_body<T, CP, KIND, BIAS>(p);
}

}  // namespace
}  // namespace sr355
