// The matrix product behind the gated feed-forward block: C[m][n] = sum over k of A[m][k] * B[n][k] on MFMA, with either
// operand stored with k contiguous ("KC": activations against weights) or with its rows contiguous ("RC": k strided, what
// the data and weight gradients read).  bf16 / fp16 on 32x32x16, fp32 on 32x32x2, fp32 accumulation.
//
// A workgroup computes BM x BN; its waves form a WM x WN grid.  A stage is 64 or 128 bytes of k per row, copied from memory
// straight into the LDS (16 bytes a lane, no registers), STAGES of them in a ring: while stage t is multiplied the next ones
// are in flight behind a counted wait, one barrier per stage.  What lies outside a matrix is read with an offset beyond the
// buffer's end, which returns zeros, so edges need no branches and every wave issues the same number of copies.
// The LDS image is permuted so that reads spread over the banks: KC tiles hold unit u (16 bytes) of row r at u ^ rot(r); RC
// tiles of 16-bit types hold each 32-byte granule at g ^ swz(k), swz even, and are read by the transposing
// ds_read_b64_tr_b16.  The copies' destination is fixed (lane order), so the permutation is applied to their sources.
// LDS reads are inline asm: a read that the compiler sees is put behind ALL copies in flight.
// The operands of the MFMA are exchanged (B first): a lane then holds four consecutive n of one m.
// Measured (bf16, 16384 x 4096 times 4096 x 1024, 256 x 256 tiles of 8 waves): 111 us = 1,240 TFLOP/s with the input in the
// last-level cache, 134 to 150 us behind the kernels that write it.  In a training step of 16384 x 1024 x 4096 the matrix pipes are
// busy 60 and 62 % of the cycles in the weight and data gradients, 47 % in this product, 37 % in gate / up and 25 % in the hidden
// gradient, whose epilogues move 0.54 and 0.67 GB with no MFMA beside them; the clock is at 1.8 to 2.0 GHz (2.6 in the launch that
// only adds).  Copies two stages further ahead took 15 % fewer cycles and 5 % less time.  Four waves of 128 x 128 (half the LDS
// reads) take the same time; two workgroups per CU on 128 x 256 (64-byte stages, half a cache line per row) 25 % more.
#pragma once
#include "token_common.h"

namespace sr355 {
namespace {

typedef void __attribute__((address_space(3))) tok_lds_void;
typedef __bf16 tok_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 tok_f16x8 __attribute__((ext_vector_type(8)));
typedef float tok_f32x4 __attribute__((ext_vector_type(4)));
typedef float tok_f32x16 __attribute__((ext_vector_type(16)));

// What the backward pass reads: act(g) and u act'(g).  fp32 is kept whole; for the 16-bit types the upper 24 bits of the
// fp32 values are kept, 16 and 8 apart.  Kept in 16 bits they put a third rounding into every gradient behind the hidden
// channels, beside those of dg / du and of the result (bf16: relative error 2.9e-3, now 2.4e-3; one rounding is 1.7e-3).
struct TokKept {
    void *a, *d;                        // [rows][h_ld] of 2 (4) bytes
    unsigned char *a_low, *d_low;       // [rows][h_ld], null for fp32
};
template <typename T>
__device__ __forceinline__ void tok_keep(void *at16, unsigned char *at8, long long at, float v) {
    if constexpr (sizeof(T) == 4) {
        ((float *)at16)[at] = v;
    } else {
        const unsigned b = __builtin_bit_cast(unsigned, v);
        ((unsigned short *)at16)[at] = (unsigned short)(b >> 16);
        at8[at] = (unsigned char)(b >> 8);
    }
}

// One product of a launch.
struct TokJob {
    const unsigned char *a[2], *b[2];   // operands of the (up to two) sections of k; GLU: b = gate and up weights
    long long a_ld, b_ld;               // bytes between rows (KC) / between k (RC)
    int M, N;
    void *c;
    long long c_ld;                     // elements
    const void *bias;                   // [N] of T, may be null
    float *part;                        // split products: [splits][M][N rounded up to 8] fp32 partials
    void *row_sums;                     // A strided in k: [M] of T, sums of A over k (may be null; c may be null with it)
    float *row_part;                    // split products: [splits][M rounded up to 8] fp32 partials of them
    int tiles_m, tiles_n;
};
struct TokGemmArgs {
    TokJob job[3];
    int first_tile[3];                  // of each job; jobs in order
    int n_jobs, n_tiles;                // n_tiles: of all jobs, one split
    int K, sections;                    // k of ONE section
    int splits, split_stages;           // stages of one split
    int act;
    const void *bias_up;                // GLU
    TokKept kept;                       // GLU: written where not null; gradient: read
    void *g, *u, *h;                    // GLU: the product (h); gradient: dg, du
    float *sums;                        // gradient: [tiles_m * WM][dg, du][N rounded up to 8], column sums of a wave's rows
    long long h_ld;                     // elements, of g / u / h / dg / du; a multiple of 16 bytes
};

enum { TOK_EPI_STORE = 0, TOK_EPI_PART = 1, TOK_EPI_GLU = 2, TOK_EPI_GLU_GRAD = 3 };

template <int BM_, int BN_, int WM_, int WN_, int KB_, int STAGES_>
struct TokTile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
    static constexpr int KB = KB_;                                  // bytes of k of a stage, 64 or 128
    static constexpr int KS = KB / 32;                              // its k steps
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int MT = BM / WM / 32, NT = BN / WN / 32;      // 32 x 32 fragments of a wave
    static constexpr int COPIES_A = BM * KB / 1024, COPIES_B = BN * KB / 1024;   // 1024-byte copies of a stage
    static constexpr int COPIES = (COPIES_A + COPIES_B) / WAVES;    // of one wave
    static constexpr int STAGE_BYTES = (BM + BN) * KB;
    static constexpr int TURN_ROW = NT * 32 * 4;                    // a row of a wave's fp32 results on their way out
    static constexpr int TURN = STAGES * STAGE_BYTES / WAVES / (32 * TURN_ROW) < MT ? STAGES * STAGE_BYTES / WAVES / (32 * TURN_ROW) : MT;
    static constexpr int LDS_BYTES = STAGES * STAGE_BYTES;
    static_assert(TURN > 0 && MT % TURN == 0, "the results turn in the stages' memory, TURN fragments at a time");
    static_assert(KS % 2 == 0, "the fragments alternate");
    static_assert(COPIES_A % WAVES == 0 && COPIES_B % WAVES == 0, "a wave's k-th copy belongs to one operand");
    static_assert(LDS_BYTES <= 160 * 1024, "LDS");
};

template <typename T>
struct TokFrag {                        // 16 bytes of k of one row: 8 (4) values
    tok_v2u lo, hi;
};

template <typename T>
__device__ __forceinline__ void tok_mfma(const tok_v4u &b, const tok_v4u &a, tok_f32x16 &c) {
    if constexpr (sizeof(T) == 4) {
        const tok_f32x4 fb = __builtin_bit_cast(tok_f32x4, b), fa = __builtin_bit_cast(tok_f32x4, a);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(fb[j], fa[j], c, 0, 0, 0);
    } else if constexpr (__is_same(T, bf16_t)) {
        c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(tok_bf16x8, b), __builtin_bit_cast(tok_bf16x8, a), c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(tok_f16x8, b), __builtin_bit_cast(tok_f16x8, a), c, 0, 0, 0);
    }
}

// Geometry of one operand's LDS image: R rows of the output side, T elements.
template <typename T, int R, int KB, bool RC>
struct TokImage {
    static constexpr int E = 16 / sizeof(T);
    static constexpr int BK = KB / sizeof(T);
    static constexpr int ROW_UNITS = KB / 16;                        // KC: units of a row
    static constexpr int K_BYTES = R * sizeof(T);                    // RC: one k of the image
    static constexpr int UNITS = K_BYTES / 16;
    static constexpr int GRANULES = K_BYTES / 32;
    static constexpr int READS = RC ? (sizeof(T) == 4 ? 4 : 2) : 1;  // LDS instructions of a fragment
    // RC: even permutation of the granules of k (16-bit types)
    static __device__ __forceinline__ int swz(int k) {
        return sizeof(T) == 4 ? 0 : (GRANULES >= 8 ? 2 * (k & 3) : (GRANULES >= 4 ? 2 * ((k >> 1) & 1) : 0));
    }
    // KC: permutation of the units of row r.  A 16-byte read goes through the 64 banks 16 lanes at a time (lanes 0-3, 12-15,
    // 20-27 and 4-11, 16-19, 28-31 of a half wave): their 16 rows then lie at 16 different places of 256 bytes.
    static __device__ __forceinline__ int rot(int r) { return ROW_UNITS == 8 ? (r >> 1) & 7 : (r >> 2) & 3; }
    // copy j of the image: the row (KC) or k (RC) that lane `lane` brings, and its unit
    static __device__ __forceinline__ void source(int j, int lane, int &line, int &unit) {
        if constexpr (!RC) {
            line = (j * 64 + lane) / ROW_UNITS;
            unit = (lane % ROW_UNITS) ^ rot(line);
        } else {
            const int at = j * 64 + lane;                            // unit of the image
            line = at / UNITS;
            const int pu = at % UNITS;
            unit = ((pu >> 1) ^ swz(line)) * 2 + (pu & 1);
        }
    }
};

__device__ __forceinline__ tok_v4u tok_join(const tok_v2u &lo, const tok_v2u &hi) { return tok_v4u{lo.x, lo.y, hi.x, hi.y}; }

// A fragment's reads.  KC: `addr` is the lane's unit, OFF the fragment's rows; RC: `addr` the lane's first piece.
template <typename T, typename I, bool RC, int OFF>
__device__ __forceinline__ void tok_read(tok_v4u &f, tok_v2u &lo, tok_v2u &hi, unsigned addr) {
    if constexpr (!RC) {
        asm volatile("ds_read_b128 %0, %1 offset:%2" : "=&v"(f) : "v"(addr), "n"(OFF) : "memory");
    } else if constexpr (sizeof(T) == 2) {
        asm volatile("ds_read_b64_tr_b16 %0, %2 offset:%3\n\tds_read_b64_tr_b16 %1, %2 offset:%4"
                     : "=&v"(lo), "=&v"(hi)
                     : "v"(addr), "n"(OFF), "n"(OFF + 4 * I::K_BYTES)
                     : "memory");
    }
}

// The activation and its derivative.  T = float goes through the exact functions, the 16-bit types through the hardware's
// exp2 and reciprocal (errors of a few 2^-23, far below their own rounding).  The normal distribution's integral is taken from
// its small side, so that gelu keeps its relative precision where it is small: fp32 by erfc, the 16-bit types as density * t P(t)
// with t = 1 / (1 + p |g|) and a polynomial of degree 6, a minimax fit that weighs the absolute error near zero and the relative one
// behind (evaluated in fp32: 1.6e-7 and, down to g = -12.9, 8e-6; half a step of fp16 is 4.9e-4).  The library's erff takes some
// 45 instructions an element, which bounded the forward pass of 262144 x 64 x 256 (130 us for the gate and up launch); this
// takes 16 and shares the exponential with the derivative.
template <bool EXACT>
__device__ __forceinline__ float tok_sigmoid(float g) {
    if constexpr (EXACT) return 1.0f / (1.0f + expf(-g));
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896f * g));
}
// the integral up to g and the density (without its 1 / sqrt(2 pi)) of the normal distribution
template <bool EXACT>
__device__ __forceinline__ void tok_normal(float g, float &cdf, float &density) {
    if constexpr (EXACT) {
        cdf = 0.5f * erfcf(-0.70710678118655f * g), density = expf(-0.5f * g * g);
    } else {
        density = __builtin_amdgcn_exp2f(-0.72134752044448f * g * g);
        const float t = __builtin_amdgcn_rcpf(1.0f + 0.347788f * fabsf(g));
        const float poly = 0.13893718f + t * (0.13539703f + t * (0.14573018f + t * (0.00086931005f + t * (0.22241315f +
                           t * (-0.18805346f + t * 0.044706643f)))));
        const float tail = t * poly * density;
        cdf = g < 0.f ? tail : 1.0f - tail;
    }
}
template <bool EXACT, int KIND>
__device__ __forceinline__ void tok_act_grad(float g, float &a, float &da) {
    if constexpr (KIND == SR355_ACT_SILU) {
        const float s = tok_sigmoid<EXACT>(g);
        a = g * s, da = s * (1.0f + g * (1.0f - s));
    } else if constexpr (KIND == SR355_ACT_GELU) {
        float cdf, density;
        tok_normal<EXACT>(g, cdf, density);
        a = g * cdf, da = cdf + g * (0.39894228040143f * density);
    } else if constexpr (KIND == SR355_ACT_RELU) {
        a = g < 0.f ? 0.f : g, da = g > 0.f ? 1.0f : 0.f;                 // (a NaN stays one)
    } else {
        a = tok_sigmoid<EXACT>(g), da = a * (1.0f - a);
    }
}
template <bool EXACT, int KIND>
__device__ __forceinline__ float tok_act(float g) {
    float a, da;
    tok_act_grad<EXACT, KIND>(g, a, da);
    return a;
}

// Eight kept values at a multiple of eight.
template <typename T>
__device__ __forceinline__ void tok_keep8(void *at16, unsigned char *at8, long long at, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; j += 4) tok_store<float, 4>((float *)at16 + at + j, *reinterpret_cast<const float(*)[4]>(v + j));
    } else {
        tok_v4u high;
        tok_v2u low;
#pragma unroll
        for (int j = 0; j < 4; ++j)                         // the upper halves of two values
            high[j] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, v[2 * j + 1]), __builtin_bit_cast(unsigned, v[2 * j]), 0x07060302u);
#pragma unroll
        for (int j = 0; j < 2; ++j)                         // byte 1 of four values
            low[j] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, v[4 * j + 1]), __builtin_bit_cast(unsigned, v[4 * j]), 0x0c0c0501u) |
                     __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, v[4 * j + 3]), __builtin_bit_cast(unsigned, v[4 * j + 2]), 0x05010c0cu);
        *reinterpret_cast<tok_v4u *>((unsigned short *)at16 + at) = high;
        *reinterpret_cast<tok_v2u *>(at8 + at) = low;
    }
}
template <typename T>
struct TokKept8 {
    tok_v4u high, more;                 // (fp32: two units)
    tok_v2u low;
    __device__ __forceinline__ void load(const void *at16, const unsigned char *at8, long long at) {
        if constexpr (sizeof(T) == 4) {
            high = *reinterpret_cast<const tok_v4u *>((const float *)at16 + at), more = *reinterpret_cast<const tok_v4u *>((const float *)at16 + at + 4);
        } else {
            high = *reinterpret_cast<const tok_v4u *>((const unsigned short *)at16 + at), low = *reinterpret_cast<const tok_v2u *>(at8 + at);
        }
    }
    __device__ __forceinline__ float value(int j) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, j < 4 ? high[j & 3] : more[j & 3]);
        return __builtin_bit_cast(float, __builtin_amdgcn_perm(high[j / 2], low[j / 4], (j & 1 ? 0x0706000cu : 0x0504000cu) | (j & 3) << 8));
    }
};

// Eight consecutive elements, in 16-byte accesses.
template <typename T>
__device__ __forceinline__ void tok_store8(T *p, const float (&v)[8]) {
    constexpr int E = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 8; j += E) tok_store<T, E>(p + j, *reinterpret_cast<const float(*)[E]>(v + j));
}
template <typename T, typename G, bool A_RC, bool B_RC, int EPI, bool SUMS>
__device__ __forceinline__ void tok_gemm_body(const TokGemmArgs &p) {
    typedef TokImage<T, G::BM, G::KB, A_RC> IA;
    typedef TokImage<T, G::BN, G::KB, B_RC> IB;
    constexpr int BK = IA::BK, E = IA::E, KS = G::KS;
    constexpr int MT = G::MT, NT = G::NT;
    constexpr unsigned OUT = 0x80000000u;                  // an offset beyond every buffer
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / G::WN, wn = wave % G::WN;

    // Workgroups go to the eight XCDs in turn: give each XCD a contiguous range of tiles, and walk a job's tiles in
    // groups of eight tile rows, so that the workgroups of one L2 share operands.
    int id = blockIdx.x;
    {
        const int n = gridDim.x, per = n / 8, extra = n % 8, xcd = id % 8, at = id / 8;
        id = xcd * per + (xcd < extra ? xcd : extra) + at;
    }
    const int split = id / p.n_tiles;
    id -= split * p.n_tiles;
    int jn = 0;
    if (p.n_jobs > 1 && id >= p.first_tile[1]) jn = 1;
    if (p.n_jobs > 2 && id >= p.first_tile[2]) jn = 2;
    const TokJob &job = p.job[jn];
    id -= p.first_tile[jn];
    constexpr int GROUP = 8;
    const int in_group = GROUP * job.tiles_n, group = id / in_group;
    const int rows_here = job.tiles_m - group * GROUP < GROUP ? job.tiles_m - group * GROUP : GROUP;
    const int tm = group * GROUP + (id - group * in_group) % rows_here, tn = (id - group * in_group) / rows_here;
    const long long m0 = (long long)tm * G::BM;
    // GLU: the tile's BN columns are BN / 2 gate columns and the up columns of the same hidden channels
    const int n0 = tn * (EPI == TOK_EPI_GLU ? G::BN / 2 : G::BN);

    // Sources of this wave's copies: byte offsets from the tile's corner, OUT where the line lies outside the matrix.
    // Copy i of the wave: image copy j = i * WAVES + wave.
    constexpr int CA = G::COPIES_A / G::WAVES, CB = G::COPIES_B / G::WAVES;
    unsigned va[CA], vb[CB];
    short ka[CA], kb[CB];                                  // first k of the copied unit, relative to the stage
#pragma unroll
    for (int i = 0; i < CA; ++i) {
        int line, unit;
        IA::source(i * G::WAVES + wave, lane, line, unit);
        if (A_RC) {
            va[i] = m0 + unit * E < job.M ? (unsigned)(line * job.a_ld + unit * 16) : OUT;
            ka[i] = line;
        } else {
            va[i] = m0 + line < job.M ? (unsigned)(line * job.a_ld + unit * 16) : OUT;
            ka[i] = unit * E;
        }
    }
#pragma unroll
    for (int i = 0; i < CB; ++i) {
        int line, unit;
        IB::source(i * G::WAVES + wave, lane, line, unit);
        if (B_RC) {
            vb[i] = n0 + unit * E < job.N ? (unsigned)(line * job.b_ld + unit * 16) : OUT;
            kb[i] = line;
        } else {
            // GLU: a wave's NT * 32 image rows are NT * 16 gate rows, then the up rows of the same hidden channels (a copy's
            // eight rows are of one kind)
            const int row = EPI == TOK_EPI_GLU ? (line / (NT * 32)) * (NT * 16) + line % (NT * 16) : line;
            vb[i] = n0 + row < job.N ? (unsigned)(row * job.b_ld + unit * 16) : OUT;
            kb[i] = unit * E;
        }
    }

    const int n_stage = (p.K + BK - 1) / BK;               // of one section
    int t0 = 0, t1 = n_stage * p.sections;
    if (EPI == TOK_EPI_PART) {
        t0 = split * p.split_stages;
        t1 = t0 + p.split_stages < t1 ? t0 + p.split_stages : t1;
    }

    // The next stage to copy: its number, operands' corners, k that is left of its section.
    const long long a_step = A_RC ? BK * job.a_ld : G::KB, b_step = B_RC ? BK * job.b_ld : G::KB;
    const long long a_corner = A_RC ? m0 * (long long)sizeof(T) : m0 * job.a_ld;
    const long long b_corner = B_RC ? n0 * (long long)sizeof(T) : n0 * job.b_ld;
    const int sec0 = EPI == TOK_EPI_PART && t0 >= n_stage ? 1 : 0, in_sec = t0 - sec0 * n_stage;   // the section of the first stage
    const unsigned char *pa = job.a[sec0] + a_corner + in_sec * a_step, *pb = job.b[sec0] + b_corner + in_sec * b_step;
    const long long up_off = job.b[1] - job.b[0];          // GLU: both weights' rows are of one stride
    const unsigned char *const pa1 = job.a[1] + a_corner, *const pb1 = job.b[1] + b_corner;
    const int sections = EPI == TOK_EPI_STORE || EPI == TOK_EPI_PART ? p.sections : 1;
    int copy_t = t0, left = p.K - in_sec * BK;
    const int K = p.K;
    // Copy I of this wave's CA + CB copies of the stage.  Past the last stage it copies zeros, so that the counted waits always
    // see the same number of copies.
    auto copy_one = [&](int slot, auto which) {
        constexpr int I = decltype(which)::value;
        const int size = copy_t < t1 ? 0x7fffffff : 0;
        unsigned char *const dst = smem + slot * G::STAGE_BYTES + wave * 1024;
        if constexpr (I < CA) {
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(pa), 0, size, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (tok_lds_void *)(dst + I * G::WAVES * 1024), 16, ka[I] < left ? va[I] : OUT, 0, 0, 0);
        } else {
            constexpr int J = I - CA;
            const unsigned char *q = pb;
            if (EPI == TOK_EPI_GLU && (((J * G::WAVES + wave) * (1024 / G::KB) / (NT * 16)) & 1)) q += up_off;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(q), 0, size, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (tok_lds_void *)(dst + G::BM * G::KB + J * G::WAVES * 1024), 16,
                                                     kb[J] < left ? vb[J] : OUT, 0, 0, 0);
        }
        if constexpr (I + 1 == CA + CB) {
            ++copy_t, left -= BK, pa += a_step, pb += b_step;
            if (sections == 2 && copy_t == n_stage) pa = pa1, pb = pb1, left = K;
        }
    };
    auto copy_stage = [&](int slot) { tok_static_for<CA + CB>([&](auto i) { copy_one(slot, i); }); };

    // Addresses of this lane's reads inside a stage.
    const unsigned lds0 = (unsigned)(size_t)(tok_lds_void *)smem;
    unsigned ra_off[A_RC ? MT : KS], rb_off[B_RC ? NT : KS];
    {
        const int half = lane >> 5, c = lane & 31;
        const int g4 = lane >> 4, q = (lane & 15) >> 2, pp = lane & 3;
        if constexpr (!A_RC) {
#pragma unroll
            for (int s = 0; s < KS; ++s) ra_off[s] = (wm * MT * 32 + c) * G::KB + (((2 * s + half) ^ IA::rot(c)) * 16);
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < MT; ++i)
                ra_off[i] = (8 * (g4 >> 1) + q) * IA::K_BYTES + ((((wm * MT + i) * 2 + (g4 & 1)) ^ IA::swz(q)) * 32) + pp * 8;
        } else {
#pragma unroll
            for (int i = 0; i < MT; ++i) ra_off[i] = 4 * half * IA::K_BYTES + ((wm * MT + i) * 32 + c) * 4;
        }
        if constexpr (!B_RC) {
#pragma unroll
            for (int s = 0; s < KS; ++s) rb_off[s] = G::BM * G::KB + (wn * NT * 32 + c) * G::KB + (((2 * s + half) ^ IB::rot(c)) * 16);
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
                rb_off[i] = G::BM * G::KB + (8 * (g4 >> 1) + q) * IB::K_BYTES + ((((wn * NT + i) * 2 + (g4 & 1)) ^ IB::swz(q)) * 32) + pp * 8;
        } else {
#pragma unroll
            for (int i = 0; i < NT; ++i) rb_off[i] = G::BM * G::KB + 4 * half * IB::K_BYTES + ((wn * NT + i) * 32 + c) * 4;
        }
    }

    tok_f32x16 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    // fragments of two k steps: the one being multiplied and the next
    // SUMS, a weight gradient: sums of A over k (a bias gradient, for which A would be read again): the waves of the first
    // column of tiles that hold its first columns add up the fragments as they pass, one lane per row and half of k.  A variant
    // of its own: the branch in the main loop costs 7 % where nothing is summed.
    // SUMS, the hidden gradient: sums of dg and du over a wave's rows, before they are rounded.
    static_assert(!SUMS || EPI == TOK_EPI_GLU_GRAD || (A_RC && (EPI == TOK_EPI_STORE || EPI == TOK_EPI_PART)), "what is summed");
    constexpr bool ROW_SUMS = SUMS && EPI != TOK_EPI_GLU_GRAD, COL_SUMS = SUMS && EPI == TOK_EPI_GLU_GRAD;
    const bool sums = ROW_SUMS && tn == 0 && wn == 0 && job.row_sums;
    float row_sum[ROW_SUMS ? MT : 1];
#pragma unroll
    for (int i = 0; i < (ROW_SUMS ? MT : 1); ++i) row_sum[i] = 0.f;
    float col_sum[COL_SUMS ? 16 : 1];                      // dg's of this lane's eight columns, then du's
#pragma unroll
    for (int i = 0; i < (COL_SUMS ? 16 : 1); ++i) col_sum[i] = 0.f;
    auto add_sums = [&](const tok_v4u (&a)[MT]) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            T v[E];
            __builtin_memcpy(v, &a[i], 16);
            float s = (float)v[0];
#pragma unroll
            for (int e = 1; e < E; ++e) s += (float)v[e];
            row_sum[i] += s;
        }
    };
    struct Frags {
        tok_v4u a[MT], b[NT];
        tok_v2u alo[MT], ahi[MT], blo[NT], bhi[NT];
        float a4[MT][4], b4[NT][4];
    } fr[2];
    // fragment X (A's, then B's) of k step S; a template, since the offsets are immediates of the instructions
    auto read_one = [&](Frags &f, unsigned base, auto step, auto which) {
        constexpr int S = decltype(step)::value;
        constexpr bool IS_A = decltype(which)::value < MT;
        constexpr int X = IS_A ? decltype(which)::value : decltype(which)::value - MT;
        typedef typename std::conditional<IS_A, IA, IB>::type I;
        constexpr bool RC = IS_A ? A_RC : B_RC;
        const unsigned *off = IS_A ? ra_off : rb_off;
        if constexpr (!RC) {
            tok_read<T, I, false, X * 32 * G::KB>(IS_A ? f.a[IS_A ? X : 0] : f.b[IS_A ? 0 : X], f.alo[0], f.ahi[0], base + off[S]);
        } else if constexpr (sizeof(T) == 2) {
            tok_v4u dummy;
            tok_read<T, I, true, S * 16 * I::K_BYTES>(dummy, IS_A ? f.alo[IS_A ? X : 0] : f.blo[IS_A ? 0 : X],
                                                      IS_A ? f.ahi[IS_A ? X : 0] : f.bhi[IS_A ? 0 : X], base + off[X]);
        } else {
            float(&v)[4] = IS_A ? f.a4[IS_A ? X : 0] : f.b4[IS_A ? 0 : X];
            asm volatile(
                "ds_read_b32 %0, %4 offset:%5\n\tds_read_b32 %1, %4 offset:%6\n\t"
                "ds_read_b32 %2, %4 offset:%7\n\tds_read_b32 %3, %4 offset:%8"
                : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
                : "v"(base + off[X]), "n"((8 * S + 0) * I::K_BYTES), "n"((8 * S + 1) * I::K_BYTES), "n"((8 * S + 2) * I::K_BYTES),
                  "n"((8 * S + 3) * I::K_BYTES)
                : "memory");
        }
    };
    // all LDS reads have returned: the fragments may be used
    auto settle = [&](Frags &f) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if constexpr (!A_RC) {
                asm volatile("" : "+v"(f.a[i]));
            } else if constexpr (sizeof(T) == 2) {
                asm volatile("" : "+v"(f.alo[i]), "+v"(f.ahi[i]));
                f.a[i] = tok_join(f.alo[i], f.ahi[i]);
            } else {
                asm volatile("" : "+v"(f.a4[i][0]), "+v"(f.a4[i][1]), "+v"(f.a4[i][2]), "+v"(f.a4[i][3]));
                f.a[i] = __builtin_bit_cast(tok_v4u, tok_f32x4{f.a4[i][0], f.a4[i][1], f.a4[i][2], f.a4[i][3]});
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if constexpr (!B_RC) {
                asm volatile("" : "+v"(f.b[i]));
            } else if constexpr (sizeof(T) == 2) {
                asm volatile("" : "+v"(f.blo[i]), "+v"(f.bhi[i]));
                f.b[i] = tok_join(f.blo[i], f.bhi[i]);
            } else {
                asm volatile("" : "+v"(f.b4[i][0]), "+v"(f.b4[i][1]), "+v"(f.b4[i][2]), "+v"(f.b4[i][3]));
                f.b[i] = __builtin_bit_cast(tok_v4u, tok_f32x4{f.b4[i][0], f.b4[i][1], f.b4[i][2], f.b4[i][3]});
            }
        }
    };

    // One wave's MFMAs of a k step leave the matrix pipe idle for every other instruction that stands between two steps, so
    // everything else stands between the MFMAs, and sched_barrier keeps it there: behind the first ones the reads of the next
    // step, behind the others copies.  In front of the first read of stage t + 1, which is in the last step of stage t,
    // stage t + 1 has to be there and every wave to be done reading stage t: a counted wait and the barrier, one per stage.
    // From there on the slot of stage t takes stage t + STAGES: a first part of the copies in that step, the rest in the
    // first step of stage t + 1.
    constexpr int MFMAS = MT * NT, READS = MT + NT;
    constexpr int FIRST_PART = (CA + CB) / 2;
    constexpr int READ_SLOTS = READS < MFMAS ? READS : MFMAS, COPY_SLOT = READ_SLOTS < MFMAS ? READ_SLOTS : 0;
#pragma unroll
    for (int s = 0; s + 1 < G::STAGES; ++s) copy_stage(s);
    tok_static_for<FIRST_PART>([&](auto i) { copy_one(G::STAGES - 1, i); });
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((G::STAGES - 2) * (CA + CB) + FIRST_PART) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    int slot = 0;
    if (t0 < t1) tok_static_for<READS>([&](auto x) { read_one(fr[0], lds0, std::integral_constant<int, 0>{}, x); });
    for (int t = t0; t < t1; ++t) {
        const unsigned base = lds0 + slot * G::STAGE_BYTES;
        const int next = slot + 1 == G::STAGES ? 0 : slot + 1, before = slot ? slot - 1 : G::STAGES - 1;
        const unsigned next_base = lds0 + next * G::STAGE_BYTES;
        tok_static_for<KS>([&](auto s) {
            constexpr int S = decltype(s)::value;
            constexpr bool LAST = S + 1 == KS;
            Frags &f = fr[S & 1];
            settle(f);
            if constexpr (LAST) {
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((G::STAGES - 2) * (CA + CB)) : "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            }
            if constexpr (ROW_SUMS) {
                if (sums) add_sums(f.a);
            }
            __builtin_amdgcn_sched_barrier(0);
            constexpr int SHARE0 = LAST ? 0 : FIRST_PART, SHARE1 = LAST ? FIRST_PART : (S == 0 ? CA + CB : FIRST_PART);
            tok_static_for<MFMAS>([&](auto mm) {
                constexpr int M = decltype(mm)::value;
                tok_mfma<T>(f.b[M % NT], f.a[M / NT], acc[M / NT][M % NT]);
                if constexpr (M < READ_SLOTS) {
                    constexpr int X0 = READS * M / READ_SLOTS, X1 = READS * (M + 1) / READ_SLOTS;
                    tok_static_for<X1 - X0>([&](auto x) {
                        // (behind the last stage: zeros that nothing uses, but the slot is there)
                        read_one(fr[(S + 1) & 1], LAST ? next_base : base, std::integral_constant<int, LAST ? 0 : S + 1>{},
                                 std::integral_constant<int, X0 + decltype(x)::value>{});
                    });
                }
                if constexpr (M >= COPY_SLOT) {
                    constexpr int A0 = SHARE0 + (SHARE1 - SHARE0) * (M - COPY_SLOT) / (MFMAS - COPY_SLOT);
                    constexpr int A1 = SHARE0 + (SHARE1 - SHARE0) * (M + 1 - COPY_SLOT) / (MFMAS - COPY_SLOT);
                    tok_static_for<A1 - A0>([&](auto x) {
                        copy_one(LAST ? slot : before, std::integral_constant<int, A0 + decltype(x)::value>{});
                    });
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        slot = next;
    }
    // the reads behind the last stage return into registers that are still theirs, and no copy may be on its way into this
    // workgroup's LDS when it is used again or ends
    settle(fr[0]);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");

    // Accumulator element e of a fragment: m = lane & 31, n = (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5).  Stored from there
    // a wave instruction would touch 32 rows, 16 bytes each; instead the wave's results turn in the LDS, TURN fragments of 32
    // rows at a time (fp32, 16-byte chunk c of row m at c ^ (m mod chunks): both directions use all banks), and every lane
    // goes on with eight consecutive columns of a row, so that memory sees whole 128-byte lines.  The rows are a loop, with
    // the activation chosen outside of it: unrolled over rows and activations the code is larger than the instruction cache
    // and its fetch took longer than the main loop (training step of 16384 x 1024 x 4096: 354 + 310 us for the two products
    // with an activation).
    constexpr bool EXACT = sizeof(T) == 4;
    if constexpr (ROW_SUMS) {
        if (sums) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const float s = row_sum[i] + __shfl_xor(row_sum[i], 32, 64);
                const long long m = m0 + (wm * MT + i) * 32 + (lane & 31);
                if (lane < 32 && m < job.M) {
                    if constexpr (EPI == TOK_EPI_PART) job.row_part[(size_t)split * ((job.M + 7) & ~7) + m] = s;
                    else ((T *)job.row_sums)[m] = (T)s;
                }
            }
        }
        if (!(EPI == TOK_EPI_PART ? (const void *)job.part : job.c)) return;
    }
    constexpr int CHUNKS = NT * 8;                          // of 4 columns
    constexpr int COLS = EPI == TOK_EPI_GLU ? NT * 16 : NT * 32;
    constexpr int LANES = COLS / 8, ROWS = 64 / LANES;      // lanes of a row, rows of an instruction
    unsigned char *const turn = smem + wave * (G::TURN * 32 * G::TURN_ROW);
    const int col = (lane % LANES) * 8;
    const int n = n0 + wn * COLS + col;
    auto turned = [&](int r, int chunk) -> tok_f32x4 {
        return *reinterpret_cast<const tok_f32x4 *>(turn + (r * CHUNKS + (chunk ^ (r % CHUNKS))) * 16);
    };
    // Results in rows of whole, aligned units go out 16 bytes a lane (all but a STORE's are laid out so, with zeros up to the
    // next eighth column); others one row of the wave's columns an instruction, one element a lane.
    constexpr int NARROW = 0, WIDE = 1;
    const bool wide = EPI != TOK_EPI_STORE || ((job.N & 7) == 0 && (job.c_ld & 7) == 0 && ((size_t)job.c & 15) == 0);
    const int n_stored = EPI == TOK_EPI_STORE ? job.N : (job.N + 7) & ~7;
    float bias[8], bias2[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        bias[j] = (EPI == TOK_EPI_GLU || EPI == TOK_EPI_STORE) && job.bias && n + j < job.N ? (float)((const T *)job.bias)[n + j] : 0.f;
        bias2[j] = EPI == TOK_EPI_GLU && p.bias_up && n + j < job.N ? (float)((const T *)p.bias_up)[n + j] : 0.f;
    }
    const bool in_n = n < n_stored;
    // Hidden channels behind the last one are stored as zeros, whatever an infinity in x or dy makes of their zero weights: they
    // are part of the units that the next product reads.
    const bool ragged = EPI == TOK_EPI_GLU || EPI == TOK_EPI_GLU_GRAD ? n + 8 > job.N : false;
    auto clear_behind = [&](float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (n + j >= job.N) v[j] = 0.f;
    };
    // rows [r of the turned fragments], all of this lane's columns
    auto finish = [&](auto kind, long long m_first) {
        constexpr int KIND = decltype(kind)::value;
        if constexpr (EPI == TOK_EPI_GLU_GRAD) {
            // UN rows' kept factors in flight: a load behind a store that it might alias waits for nothing else, but is not
            // moved in front of it
            constexpr int UN = G::TURN * 32 / ROWS < 8 ? G::TURN * 32 / ROWS : 8;
            static_assert(G::TURN * 32 % (ROWS * UN) == 0, "whole groups of rows");
            for (int r0 = lane / LANES; r0 < G::TURN * 32; r0 += ROWS * UN) {
                TokKept8<T> ka[UN], kd[UN];
#pragma unroll
                for (int k = 0; k < UN; ++k) {
                    const long long m = m_first + r0 + k * ROWS;
                    if (m >= job.M || !in_n) continue;
                    ka[k].load(p.kept.a, p.kept.a_low, m * p.h_ld + n);
                    kd[k].load(p.kept.d, p.kept.d_low, m * p.h_ld + n);
                }
#pragma unroll
                for (int k = 0; k < UN; ++k) {
                    const int r = r0 + k * ROWS;
                    const long long m = m_first + r;
                    if (m >= job.M || !in_n) continue;
                    const tok_f32x4 lo = turned(r, col / 4), hi = turned(r, col / 4 + 1);
                    const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                    float dg[8], du[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) dg[j] = v[j] * kd[k].value(j), du[j] = v[j] * ka[k].value(j);
                    if (ragged) clear_behind(dg), clear_behind(du);
                    if constexpr (COL_SUMS) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) col_sum[j] += dg[j], col_sum[8 + j] += du[j];
                    }
                    tok_store8<T>((T *)p.g + m * p.h_ld + n, dg);
                    tok_store8<T>((T *)p.u + m * p.h_ld + n, du);
                }
            }
            return;
        }
        if constexpr (EPI == TOK_EPI_STORE && KIND == NARROW) {
            static_assert(COLS == 64, "a lane per column");
            const int n1 = n0 + wn * COLS + lane;
            if (n1 >= job.N) return;
            const float b = job.bias ? (float)((const T *)job.bias)[n1] : 0.f;
            const int rows = job.M - m_first < G::TURN * 32 ? (int)(job.M - m_first) : G::TURN * 32;
            T *c = (T *)job.c + m_first * job.c_ld + n1;
#pragma unroll 4
            for (int r = 0; r < rows; ++r) c[r * job.c_ld] = (T)(turned(r, lane / 4)[lane & 3] + b);
            return;
        }
#pragma unroll 2
        for (int r = lane / LANES; r < G::TURN * 32; r += ROWS) {
            const long long m = m_first + r;
            const tok_f32x4 lo = turned(r, col / 4), hi = turned(r, col / 4 + 1);
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (m >= job.M || !in_n) continue;
            if constexpr (EPI == TOK_EPI_GLU) {
                const tok_f32x4 lo2 = turned(r, NT * 4 + col / 4), hi2 = turned(r, NT * 4 + col / 4 + 1);
                float w[8] = {lo2[0], lo2[1], lo2[2], lo2[3], hi2[0], hi2[1], hi2[2], hi2[3]}, h[8];
                const long long at = m * p.h_ld + n;
                if (p.kept.a) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float up = w[j] + bias2[j];
                        float da;
                        tok_act_grad<EXACT, KIND>(v[j] + bias[j], v[j], da);
                        h[j] = v[j] * up, w[j] = up * da;
                    }
                    if (ragged) clear_behind(v), clear_behind(w), clear_behind(h);
                    tok_keep8<T>(p.kept.a, p.kept.a_low, at, v);
                    tok_keep8<T>(p.kept.d, p.kept.d_low, at, w);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[j] = tok_act<EXACT, KIND>(v[j] + bias[j]) * (w[j] + bias2[j]);
                    if (ragged) clear_behind(h);
                }
                tok_store8<T>((T *)p.h + at, h);
            } else if constexpr (EPI == TOK_EPI_PART) {
                tok_store8<float>(job.part + ((size_t)split * job.M + m) * n_stored + n, v);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += bias[j];
                tok_store8<T>((T *)job.c + m * job.c_ld + n, v);
            }
        }
    };
#pragma unroll
    for (int i0 = 0; i0 < MT; i0 += G::TURN) {
        asm volatile("" ::: "memory");                      // (the lanes of a wave read what others of them wrote, in order)
#pragma unroll
        for (int i = 0; i < G::TURN; ++i) {
            const int r0 = i * 32 + (lane & 31);
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int chunk = j * 8 + q * 2 + (lane >> 5);
                    const tok_f32x16 &a = acc[i0 + i][j];
                    *reinterpret_cast<tok_f32x4 *>(turn + (r0 * CHUNKS + (chunk ^ (r0 % CHUNKS))) * 16) =
                        tok_f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
                }
        }
        asm volatile("" ::: "memory");
        const long long m_first = m0 + (wm * MT + i0) * 32;
        if constexpr (EPI == TOK_EPI_GLU) {
            if (p.act == SR355_ACT_SILU) finish(std::integral_constant<int, SR355_ACT_SILU>{}, m_first);
            else if (p.act == SR355_ACT_GELU) finish(std::integral_constant<int, SR355_ACT_GELU>{}, m_first);
            else if (p.act == SR355_ACT_RELU) finish(std::integral_constant<int, SR355_ACT_RELU>{}, m_first);
            else finish(std::integral_constant<int, SR355_ACT_SIGMOID>{}, m_first);
        } else {
            if (wide) finish(std::integral_constant<int, WIDE>{}, m_first);
            else finish(std::integral_constant<int, NARROW>{}, m_first);
        }
    }
    if constexpr (COL_SUMS) {
        // the lanes that hold the same columns, in a fixed order
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int o = LANES; o < 64; o <<= 1) col_sum[j] += __shfl_xor(col_sum[j], o, 64);
        if (lane < LANES && in_n) {
            float *part = p.sums + ((size_t)tm * G::WM + wm) * 2 * n_stored + n;
            tok_store8<float>(part, *reinterpret_cast<const float(*)[8]>(col_sum));
            tok_store8<float>(part + n_stored, *reinterpret_cast<const float(*)[8]>(col_sum + 8));
        }
    }
}

template <typename T, typename G, bool A_RC, bool B_RC, int EPI, bool SUMS = false>
__global__ __launch_bounds__(G::THREADS) void tok_gemm_kernel(TokGemmArgs p) {
    tok_gemm_body<T, G, A_RC, B_RC, EPI, SUMS>(p);
}

}  // namespace
}  // namespace sr355
