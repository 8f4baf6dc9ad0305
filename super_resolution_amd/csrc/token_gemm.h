// The matrix product behind the gated feed-forward block: C[m][n] = sum over k of A[m][k] * B[n][k] on MFMA, with either
// operand stored with k contiguous ("KC": activations against weights) or with its rows contiguous ("RC": k strided, what
// the data and weight gradients read).  bf16 / fp16 on 32x32x16, fp32 on 32x32x2, fp32 accumulation.
//
// A workgroup computes BM x BN; its waves form a WM x WN grid.  A stage is 128 bytes of k per row, copied from memory
// straight into the LDS (16 bytes a lane, no registers), STAGES of them in a ring: while stage t is multiplied the next
// ones are in flight behind a counted wait, one barrier per stage.  What lies outside a matrix is read with an offset
// beyond the buffer's end, which returns zeros, so edges need no branches and every wave issues the same number of copies.
// The LDS image is permuted so that reads spread over the banks: KC tiles (rows of 8 units of 16 bytes) hold unit u of row
// r at u ^ (r & 7); RC tiles of 16-bit types hold each 32-byte granule at g ^ f(k), f even, and are read by the transposing
// ds_read_b64_tr_b16.  The copies' destination is fixed (lane order), so the permutation is applied to their sources.
// LDS reads are inline asm: a read that the compiler sees is put behind ALL copies in flight.  The reads of one k step are
// issued before the MFMAs of the step in front of it and waited for by count.
// The operands of the MFMA are exchanged (B first): a lane then holds four consecutive n of one m, what a row-major store
// wants.
#pragma once
#include "token_common.h"

namespace sr355 {
namespace {

typedef void __attribute__((address_space(3))) tok_lds_void;
typedef __bf16 tok_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 tok_f16x8 __attribute__((ext_vector_type(8)));
typedef float tok_f32x4 __attribute__((ext_vector_type(4)));
typedef float tok_f32x16 __attribute__((ext_vector_type(16)));

// One product of a launch.
struct TokJob {
    const unsigned char *a[2], *b[2];   // operands of the (up to two) sections of k; GLU: b = gate and up weights
    long long a_ld, b_ld;               // bytes between rows (KC) / between k (RC)
    int M, N;
    void *c;
    long long c_ld;                     // elements
    const void *bias;                   // [N] of T, may be null
    float *part;                        // split products: [splits][M][N] fp32 partials
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
    void *g, *u, *h;                    // GLU: saved (may be null) and product; gradient: dg, du (in g, u)
    const void *sg, *su;                // gradient: saved g and u
    long long h_ld;                     // elements, of g / u / h / dg / du; a multiple of 16 bytes
};

enum { TOK_EPI_STORE = 0, TOK_EPI_PART = 1, TOK_EPI_GLU = 2, TOK_EPI_GLU_GRAD = 3 };

template <int BM_, int BN_, int WM_, int WN_, int STAGES_>
struct TokTile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_;
    static constexpr int WAVES = WM * WN, THREADS = 64 * WAVES;
    static constexpr int MT = BM / WM / 32, NT = BN / WN / 32;      // 32 x 32 fragments of a wave
    static constexpr int COPIES_A = BM / 8, COPIES_B = BN / 8;      // 1024-byte copies of a stage
    static constexpr int COPIES = (COPIES_A + COPIES_B) / WAVES;    // of one wave
    static constexpr int STAGE_BYTES = (BM + BN) * 128;
    static constexpr int LDS_BYTES = STAGES * STAGE_BYTES;
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
template <typename T, int R, bool RC>
struct TokImage {
    static constexpr int E = 16 / sizeof(T);
    static constexpr int BK = 128 / sizeof(T);
    static constexpr int K_BYTES = R * sizeof(T);                    // RC: one k of the image
    static constexpr int UNITS = K_BYTES / 16;
    static constexpr int GRANULES = K_BYTES / 32;
    static constexpr int READS = RC ? (sizeof(T) == 4 ? 4 : 2) : 1;  // LDS instructions of a fragment
    // RC: even permutation of the granules of k (16-bit types)
    static __device__ __forceinline__ int swz(int k) {
        return sizeof(T) == 4 ? 0 : (GRANULES >= 8 ? 2 * (k & 3) : (GRANULES >= 4 ? 2 * ((k >> 1) & 1) : 0));
    }
    // copy j of the image: the row (KC) or k (RC) that lane `lane` brings, and its unit
    static __device__ __forceinline__ void source(int j, int lane, int &line, int &unit) {
        if constexpr (!RC) {
            line = 8 * j + (lane >> 3);
            unit = (lane & 7) ^ (lane >> 3);
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
// exp2 and reciprocal (errors of a few 2^-23, far below their own rounding).
template <bool EXACT>
__device__ __forceinline__ float tok_sigmoid(float g) {
    if constexpr (EXACT) return 1.0f / (1.0f + expf(-g));
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896f * g));
}
template <bool EXACT>
__device__ __forceinline__ float tok_gauss(float g) {      // exp(-g^2 / 2)
    if constexpr (EXACT) return expf(-0.5f * g * g);
    return __builtin_amdgcn_exp2f(-0.72134752044448f * g * g);
}
template <bool EXACT>
__device__ __forceinline__ float tok_act(int kind, float g) {
    if (kind == SR355_ACT_SILU) return g * tok_sigmoid<EXACT>(g);
    if (kind == SR355_ACT_GELU) return g * (0.5f * (1.0f + erff(0.70710678118655f * g)));
    if (kind == SR355_ACT_RELU) return g < 0.f ? 0.f : g;             // (a NaN stays one)
    return tok_sigmoid<EXACT>(g);
}
template <bool EXACT>
__device__ __forceinline__ void tok_act_grad(int kind, float g, float &a, float &da) {
    if (kind == SR355_ACT_SILU) {
        const float s = tok_sigmoid<EXACT>(g);
        a = g * s, da = s * (1.0f + g * (1.0f - s));
    } else if (kind == SR355_ACT_GELU) {
        const float cdf = 0.5f * (1.0f + erff(0.70710678118655f * g));
        a = g * cdf, da = cdf + g * (0.39894228040143f * tok_gauss<EXACT>(g));
    } else if (kind == SR355_ACT_RELU) {
        a = g < 0.f ? 0.f : g, da = g > 0.f ? 1.0f : 0.f;
    } else {
        a = tok_sigmoid<EXACT>(g), da = a * (1.0f - a);
    }
}

// Four consecutive elements.
template <typename T>
__device__ __forceinline__ void tok_store4(T *p, const float (&v)[4]) {
    T t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = (T)v[j];
    if constexpr (sizeof(T) == 2) {
        tok_v2u raw;
        __builtin_memcpy(&raw, t, 8);
        *reinterpret_cast<tok_v2u *>(p) = raw;
    } else {
        tok_v4u raw;
        __builtin_memcpy(&raw, t, 16);
        *reinterpret_cast<tok_v4u *>(p) = raw;
    }
}
template <typename T>
__device__ __forceinline__ void tok_load4(const T *p, float (&v)[4]) {
    T t[4];
    if constexpr (sizeof(T) == 2) {
        const tok_v2u raw = *reinterpret_cast<const tok_v2u *>(p);
        __builtin_memcpy(t, &raw, 8);
    } else {
        const tok_v4u raw = *reinterpret_cast<const tok_v4u *>(p);
        __builtin_memcpy(t, &raw, 16);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)t[j];
}

template <typename T, typename G, bool A_RC, bool B_RC, int EPI>
__device__ __forceinline__ void tok_gemm_body(const TokGemmArgs &p) {
    typedef TokImage<T, G::BM, A_RC> IA;
    typedef TokImage<T, G::BN, B_RC> IB;
    constexpr int BK = IA::BK, E = IA::E, KS = 4;          // four k steps of 32 bytes per stage
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
            // GLU: blocks of 64 image rows = 32 gate rows, then 32 up rows (a copy's eight rows are of one kind)
            const int row = EPI == TOK_EPI_GLU ? (line >> 6) * 32 + (line & 31) : line;
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

    auto copy_stage = [&](int t, int slot) {
        const bool live = t < t1;
        const int sec = t >= n_stage ? 1 : 0;
        const int k0 = (t - sec * n_stage) * BK;
        const unsigned char *pa = job.a[EPI == TOK_EPI_GLU ? 0 : sec], *pb = job.b[EPI == TOK_EPI_GLU ? 0 : sec];
        const long long ao = A_RC ? k0 * job.a_ld + m0 * (long long)sizeof(T) : m0 * job.a_ld + k0 * (long long)sizeof(T);
        const long long bo = B_RC ? k0 * job.b_ld + n0 * (long long)sizeof(T) : n0 * job.b_ld + k0 * (long long)sizeof(T);
        const int size = live ? 0x7fffffff : 0;
        __amdgpu_buffer_rsrc_t ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(pa + ao), 0, size, 0x00020000);
        __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(pb + bo), 0, size, 0x00020000);
        __amdgpu_buffer_rsrc_t rb2 = rb;
        if (EPI == TOK_EPI_GLU)
            rb2 = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char *>(job.b[1] + bo), 0, size, 0x00020000);
        unsigned char *dst = smem + slot * G::STAGE_BYTES + wave * 1024;
        const int left = p.K - k0;
        if (left >= BK) {
#pragma unroll
            for (int i = 0; i < CA; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (tok_lds_void *)(dst + i * G::WAVES * 1024), 16, va[i], 0, 0, 0);
#pragma unroll
            for (int i = 0; i < CB; ++i) {
                const bool up = EPI == TOK_EPI_GLU && (((i * G::WAVES + wave) >> 2) & 1);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(up ? rb2 : rb, (tok_lds_void *)(dst + G::BM * 128 + i * G::WAVES * 1024), 16,
                                                         vb[i], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < CA; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (tok_lds_void *)(dst + i * G::WAVES * 1024), 16,
                                                         ka[i] < left ? va[i] : OUT, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < CB; ++i) {
                const bool up = EPI == TOK_EPI_GLU && (((i * G::WAVES + wave) >> 2) & 1);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(up ? rb2 : rb, (tok_lds_void *)(dst + G::BM * 128 + i * G::WAVES * 1024), 16,
                                                         kb[i] < left ? vb[i] : OUT, 0, 0, 0);
            }
        }
    };

    // Addresses of this lane's reads inside a stage.
    const unsigned lds0 = (unsigned)(size_t)(tok_lds_void *)smem;
    unsigned ra_off[A_RC ? MT : KS], rb_off[B_RC ? NT : KS];
    {
        const int half = lane >> 5, c = lane & 31;
        const int g4 = lane >> 4, q = (lane & 15) >> 2, pp = lane & 3;
        if constexpr (!A_RC) {
#pragma unroll
            for (int s = 0; s < KS; ++s) ra_off[s] = (wm * MT * 32 + c) * 128 + (((2 * s + half) ^ (c & 7)) * 16);
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
            for (int s = 0; s < KS; ++s) rb_off[s] = G::BM * 128 + (wn * NT * 32 + c) * 128 + (((2 * s + half) ^ (c & 7)) * 16);
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < NT; ++i)
                rb_off[i] = G::BM * 128 + (8 * (g4 >> 1) + q) * IB::K_BYTES + ((((wn * NT + i) * 2 + (g4 & 1)) ^ IB::swz(q)) * 32) + pp * 8;
        } else {
#pragma unroll
            for (int i = 0; i < NT; ++i) rb_off[i] = G::BM * 128 + 4 * half * IB::K_BYTES + ((wn * NT + i) * 32 + c) * 4;
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
    struct Frags {
        tok_v4u a[MT], b[NT];
        tok_v2u alo[MT], ahi[MT], blo[NT], bhi[NT];
        float a4[MT][4], b4[NT][4];
    } fr[2];
    auto read_step = [&](Frags &f, unsigned base, auto step) {
        constexpr int S = decltype(step)::value;
        // (a template loop: the offsets are immediates of the instructions)
        auto one = [&](auto which, auto index) {
            constexpr bool IS_A = decltype(which)::value == 0;
            constexpr int X = decltype(index)::value;
            typedef typename std::conditional<IS_A, IA, IB>::type I;
            constexpr bool RC = IS_A ? A_RC : B_RC;
            const unsigned *off = IS_A ? ra_off : rb_off;
            if constexpr (!RC) {
                tok_read<T, I, false, X * 32 * 128>(IS_A ? f.a[IS_A ? X : 0] : f.b[IS_A ? 0 : X], f.alo[0], f.ahi[0], base + off[S]);
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
        tok_static_for<MT>([&](auto i) { one(std::integral_constant<int, 0>{}, i); });
        tok_static_for<NT>([&](auto i) { one(std::integral_constant<int, 1>{}, i); });
    };
    // at most PENDING younger LDS instructions outstanding, then the fragments may be used
    constexpr int STEP_READS = MT * IA::READS + NT * IB::READS;
    auto settle = [&](Frags &f, auto pending) {
        constexpr int P = decltype(pending)::value < 15 ? decltype(pending)::value : 15;
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(P) : "memory");
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
    auto multiply = [&](const Frags &f) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) tok_mfma<T>(f.b[j], f.a[i], acc[i][j]);
    };

    constexpr int AHEAD = G::STAGES - 1;
#pragma unroll
    for (int s = 0; s < AHEAD; ++s) copy_stage(t0 + s, s);
    int slot = 0;
    for (int t = t0; t < t1; ++t) {
        // stage t has landed once at most the copies of the AHEAD - 1 younger stages are outstanding; past the barrier it
        // has for every wave, and every wave has left the slot of stage t - 1
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"((AHEAD - 1) * (CA + CB)) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const int next = slot + AHEAD >= G::STAGES ? slot + AHEAD - G::STAGES : slot + AHEAD;
        copy_stage(t + AHEAD, next);
        const unsigned base = lds0 + slot * G::STAGE_BYTES;
        read_step(fr[0], base, std::integral_constant<int, 0>{});
        tok_static_for<KS>([&](auto s) {
            constexpr int S = decltype(s)::value;
            if constexpr (S + 1 < KS) {
                read_step(fr[(S + 1) & 1], base, std::integral_constant<int, S + 1>{});
                settle(fr[S & 1], std::integral_constant<int, STEP_READS>{});
            } else {
                settle(fr[S & 1], std::integral_constant<int, 0>{});
            }
            multiply(fr[S & 1]);
        });
        slot = slot + 1 == G::STAGES ? 0 : slot + 1;
    }
    // no copy may still be on its way into this workgroup's LDS when it ends
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    // Accumulator element e of a fragment: m = lane & 31, n = (e & 3) + 8 * (e >> 2) + 4 * (lane >> 5).
    constexpr bool EXACT = sizeof(T) == 4;
    const int half4 = 4 * (lane >> 5);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long long m = m0 + (wm * MT + i) * 32 + (lane & 31);
        if (m >= job.M) continue;
        if constexpr (EPI == TOK_EPI_GLU) {
            static_assert(NT == 2, "a wave holds the gate and the up columns of 32 hidden channels");
            const int nb = n0 + wn * 32 + half4;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = nb + 8 * q;
                if (n >= p.h_ld) continue;
                float g4[4], u4[4], h4[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // columns past the hidden width (up to the padded row) have zero products and no bias: they store zeros
                    g4[j] = acc[i][0][4 * q + j], u4[j] = acc[i][NT - 1][4 * q + j];
                    if (job.bias && n + j < job.N) g4[j] += (float)((const T *)job.bias)[n + j];
                    if (p.bias_up && n + j < job.N) u4[j] += (float)((const T *)p.bias_up)[n + j];
                    h4[j] = tok_act<EXACT>(p.act, g4[j]) * u4[j];
                }
                const long long at = m * p.h_ld + n;
                tok_store4<T>((T *)p.h + at, h4);
                if (p.g) {
                    tok_store4<T>((T *)p.g + at, g4);
                    tok_store4<T>((T *)p.u + at, u4);
                }
            }
        } else {
#pragma unroll
            for (int jn2 = 0; jn2 < NT; ++jn2) {
                const int nb = n0 + (wn * NT + jn2) * 32 + half4;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int n = nb + 8 * q;
                    float v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = acc[i][jn2][4 * q + j];
                    if constexpr (EPI == TOK_EPI_GLU_GRAD) {
                        if (n >= p.h_ld) continue;
                        const long long at = m * p.h_ld + n;
                        float g4[4], u4[4], dg[4], du[4];
                        tok_load4<T>((const T *)p.sg + at, g4);
                        tok_load4<T>((const T *)p.su + at, u4);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float act, da;
                            tok_act_grad<EXACT>(p.act, g4[j], act, da);
                            dg[j] = v[j] * u4[j] * da, du[j] = v[j] * act;
                        }
                        tok_store4<T>((T *)p.g + at, dg);
                        tok_store4<T>((T *)p.u + at, du);
                    } else if constexpr (EPI == TOK_EPI_PART) {
                        if (n >= job.N) continue;
                        float *part = job.part + ((size_t)split * job.M + m) * job.N + n;
                        if ((job.N & 3) == 0) {
                            tok_store4<float>(part, v);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (n + j < job.N) part[j] = v[j];
                        }
                    } else {
                        if (n >= job.N) continue;
                        if (job.bias) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (n + j < job.N) v[j] += (float)((const T *)job.bias)[n + j];
                        }
                        T *c = (T *)job.c + m * job.c_ld + n;
                        if ((job.N & 3) == 0 && (job.c_ld & 3) == 0 && ((size_t)job.c & 15) == 0) {
                            tok_store4<T>(c, v);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                if (n + j < job.N) c[j] = (T)v[j];
                        }
                    }
                }
            }
        }
    }
}

template <typename T, typename G, bool A_RC, bool B_RC, int EPI>
__global__ __launch_bounds__(G::THREADS) void tok_gemm_kernel(TokGemmArgs p) {
    tok_gemm_body<T, G, A_RC, B_RC, EPI>(p);
}

}  // namespace
}  // namespace sr355
