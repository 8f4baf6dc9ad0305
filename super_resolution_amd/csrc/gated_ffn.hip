// The gated feed-forward block on rows of channels and its gradients:
//     g = x Wg' + bg, u = x Wu' + bu, h = act(g) * u, y = h Wd' + bd;
//     dh = dy Wd, dg = dh * u * act'(g), du = dh * act(g), dx = dg Wg + du Wu,
//     dWg = dg' x, dWu = du' x, dWd = dy' h, biases: column sums of dg, du, dy.
// Forward: one launch computes both projections, the activation and the product (a workgroup multiplies its rows of x with
// the gate and the up weights of the same hidden channels, so g and u meet in a wave's registers), one the projection back.
// Training keeps act(g), u act'(g) and h, inference h alone.  Backward: one launch computes dh and, in its epilogue, dg and
// du (two products per element: the derivative is taken in the forward pass, from g and u as they were accumulated); one dx,
// over both sections of k; one all three weight gradients and w_down's bias gradient.  Products accumulate in fp32.  Between
// the launches h, dg and du are held in the type of x, to which they are rounded as operands of products in any case; the other
// two bias gradients are summed before that rounding, in the epilogue and one more launch.
//
// Operands are read 16 bytes at a time.  What does not allow that (a width, stride or pointer that is no multiple of 16
// bytes) is first copied into padded rows of the workspace, one launch for all of them.
#include <climits>

#include "token_narrow.h"
#include "token_rows.h"

namespace sr355 {

namespace {
// 16-bit types: 256 x 256 tiles, one workgroup per CU, or 128 x 128, two per CU (tiles_are_big).  A row's share of a stage is a
// whole 128-byte line where k is contiguous (with 64 bytes every line comes twice from the L2: 147 against 138 us for
// 16384 x 4096 times 4096 x 1024); where k is strided a stage's rows are lines in any case, and five stages of 64 bytes hide
// more latency than two of 128 (443 against 472 us for the three weight gradients of 16384 x 1024 x 4096).
typedef TokTile<256, 256, 2, 4, 128, 2> Tile256;
typedef TokTile<256, 256, 2, 4, 64, 5> TileWgrad;
typedef TokTile<128, 128, 2, 2, 128, 2> Tile128;
// As many small tiles as CUs or fewer: one per CU, so the ring may take three stages (bf16, gate / up of 65 rows, 2048 x 8192:
// 22 against 27 us, 1024 x 4096: 15 against 17, of 200 rows 26 against 30; four stages take no less).
typedef TokTile<128, 128, 2, 2, 128, 3> TileFew;
constexpr int N_CU = 256;

// fp32: 32 x 32 x 2 instructions take eight times as long for the same bytes, so operand traffic does not matter and small tiles,
// three workgroups per CU, hide starts and ends best (forward and backward kernels, 1000 x 256 x 1024: 102 us, with 128 x 128
// tiles, two per CU, 128; 3001 x 501 x 1333: 438 and 474; 9000 x 1024 x 4096: 5473 and 5593, with 256 x 256 tiles 6502).
typedef TokTile<128, 64, 4, 1, 128, 2> TileF32;
template <typename T>
using TileSmall = typename std::conditional<sizeof(T) == 4, TileF32, Tile128>::type;
struct SmallShape {
    int bm, bn, kb, slots;       // slots: workgroups of all CUs at a time
    SmallShape(int dtype) {
        if (dtype == SR355_DTYPE_F32) bm = TileF32::BM, bn = TileF32::BN, kb = TileF32::KB, slots = 3 * N_CU;
        else bm = Tile128::BM, bn = Tile128::BN, kb = Tile128::KB, slots = 2 * N_CU;
    }
    long long tiles(long long m, long long n) const { return tok_cdiv(m, bm) * tok_cdiv(n, bn); }
};

struct PadJob {
    const void *src;
    void *dst;
    long long rows, src_ld, dst_ld;   // elements
    int cols;
};
struct PadArgs {
    PadJob job[6];
};
// Rows of `cols` elements into rows of dst_ld (whole units), zeros behind.  Neither side of an odd row is aligned to more than
// an element, so a wave moves 64 neighbouring elements an instruction, eight of them in flight.
template <typename T>
__global__ __launch_bounds__(256) void pad_rows_kernel(PadArgs p) {
    constexpr int UN = 8;
    const PadJob &j = p.job[blockIdx.y];
    const int lane = threadIdx.x & 63;
    const long long per_row = (j.dst_ld + 64 * UN - 1) / (64 * UN), n = j.rows * per_row;
    for (long long i = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); i < n; i += (long long)gridDim.x * 4) {
        const long long row = i / per_row;
        const int c0 = (int)(i - row * per_row) * 64 * UN + lane;
        const T *src = (const T *)j.src + row * j.src_ld;
        T *dst = (T *)j.dst + row * j.dst_ld, v[UN];
#pragma unroll
        for (int k = 0; k < UN; ++k) v[k] = c0 + k * 64 < j.cols ? src[c0 + k * 64] : (T)0.f;
#pragma unroll
        for (int k = 0; k < UN; ++k)
            if (c0 + k * 64 < j.dst_ld) dst[c0 + k * 64] = v[k];
    }
}

// out[row][col] = sum over splits, in order, of part[s][row][col]; rows of the parts are whole groups of eight columns
struct ReduceJob {
    const float *part;
    void *out;
    long long rows;
    int cols;
};
struct ReduceArgs {
    ReduceJob job[6];
    int splits;
    const void *bias;        // of columns, may be null
};
template <typename T>
__global__ __launch_bounds__(256) void reduce_splits_kernel(ReduceArgs a) {
    const ReduceJob &job = a.job[blockIdx.y];
    const float *part = job.part;
    const int cols = job.cols, ld = (cols + 7) & ~7;
    const long long n = job.rows * ld;
    const bool vec = cols == ld && ((size_t)job.out & 15) == 0;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (long long)gridDim.x * 1024) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        // eight parts in flight (one after the other 32 parts of a small product took 10 us)
        for (int s = 0; s < a.splits; s += 8) {
            float t[8][4];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
#pragma unroll
                for (int j = 0; j < 4; ++j) t[k][j] = 0.f;
                if (s + k < a.splits) tok_load<float, 4>(part + (size_t)(s + k) * n + i, t[k]);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += t[k][j];
        }
        const long long row = n <= 0x7fffffff ? (unsigned)i / (unsigned)ld : i / ld;
        const int col = (int)(i - row * ld);
        T *out = (T *)job.out + row * cols + col;
        T o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = (T)(v[j] + (a.bias && col + j < cols ? (float)((const T *)a.bias)[col + j] : 0.f));
        if (vec) {
            __builtin_memcpy(__builtin_assume_aligned(out, 4 * sizeof(T)), o, 4 * sizeof(T));
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < cols) out[j] = o[j];
        }
    }
}

template <typename T, typename G, bool A_RC, bool B_RC, int EPI, bool SUMS = false>
int gemm_launch(const TokGemmArgs &g, const char *what, hipStream_t stream) {
    // (a grid axis holds fewer than 2^32 threads; the runtime drops more without an error)
    if ((long long)g.n_tiles * g.splits * G::THREADS > 0xffffffffLL) {
        set_error("%s: too many tiles for one launch", what);
        return SR355_ERR_INVALID;
    }
    void (*const kernel)(TokGemmArgs) = tok_gemm_kernel<T, G, A_RC, B_RC, EPI, SUMS>;
    if (G::LDS_BYTES > 64 * 1024) {
        // (per device, and cheap: not remembered)
        const hipError_t e = hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, G::LDS_BYTES);
        if (e != hipSuccess) return check_hip(e, what);
    }
    hipLaunchKernelGGL(kernel, dim3((unsigned)(g.n_tiles * g.splits)), dim3(G::THREADS), G::LDS_BYTES, stream, g);
    return check_hip(hipGetLastError(), what);
}

template <typename G>
long long set_tiles(TokGemmArgs &g, bool glu) {
    long long n = 0;
    for (int j = 0; j < g.n_jobs; ++j) {
        g.first_tile[j] = (int)n;
        g.job[j].tiles_m = (int)tok_cdiv(g.job[j].M, G::BM);
        g.job[j].tiles_n = (int)tok_cdiv(g.job[j].N, glu ? G::BN / 2 : G::BN);
        n += (long long)g.job[j].tiles_m * g.job[j].tiles_n;
    }
    g.n_tiles = (int)(n < INT_MAX ? n : INT_MAX);
    return n;
}

// Which tiles take less: a CU works on one big or two small ones at a time, a quarter as much work each, and a round of big
// ones takes 0.85 of two rounds of small ones for the halved operand traffic (bf16, 1024 x 4096, gate / up, big against small
// tiles: 1500 rows 35 against 39 us, 4096 rows 83 against 98, 12000 rows 255 against 304).  What decides else is how full the
// last round is (3000 rows, 384 big or 1536 small tiles: 70 against 67; down of 20000 rows, 316 or 1256: 235 against 219).
bool tiles_are_big(long long big, long long small) { return 1.7 * tok_cdiv(big, N_CU) <= tok_cdiv(small, 2 * N_CU); }

template <typename T, bool A_RC, bool B_RC, int EPI, bool SUMS = false>
int gemm_pick(TokGemmArgs &g, const char *what, hipStream_t stream) {
    g.splits = 1;
    const bool glu = EPI == TOK_EPI_GLU;
    if constexpr (sizeof(T) == 2) {
        const long long small = set_tiles<Tile128>(g, glu);
        if (small <= N_CU) return gemm_launch<T, TileFew, A_RC, B_RC, EPI, SUMS>(g, what, stream);
        if (tiles_are_big(set_tiles<Tile256>(g, glu), small)) return gemm_launch<T, Tile256, A_RC, B_RC, EPI, SUMS>(g, what, stream);
    }
    set_tiles<TileSmall<T>>(g, glu);
    return gemm_launch<T, TileSmall<T>, A_RC, B_RC, EPI, SUMS>(g, what, stream);
}

// Into how many parts the sum over k of a few tiles is split: the number that takes least, by the rounds of the chip
// (`slots` workgroups at a time) and the partials' way through memory (8 bytes an element and part at 5 TB/s, and a launch).
// Microseconds of a stage, with as many workgroups per CU as fit: what the kernels take on full rounds.
struct Splits {
    int n, stages;      // parts, stages of a part
};
Splits pick_splits(long long tiles, int slots, long long stages, double elements, double stage_us) {
    if (stages < 1) stages = 1;
    Splits best = {1, (int)stages};
    double least = 1e30;
    for (long long s = 1; s <= 64 && s <= (stages + 3) / 4; ++s) {
        const long long per = tok_cdiv(stages, s), n = tok_cdiv(stages, per);
        const double us = (double)tok_cdiv(tiles * n, slots) * per * stage_us + (n > 1 ? 4.0 + 8e-6 / 5.0 * n * elements : 0.0);
        if (us < least) least = us, best = {(int)n, (int)per};
    }
    return best;
}
template <typename G>
double stage_us(int dtype) {
    // MFMA cycles of a stage's workgroups on a CU (32 a 32 x 32 x 16, 64 a 32 x 32 x 2) at 2 GHz and 70 % of the pipes
    const double wgs = 160 * 1024 / G::LDS_BYTES;
    const double mfma = (double)G::MT * G::NT * G::KS * (dtype == SR355_DTYPE_F32 ? 4 * 64 : 32) * (G::WAVES / 4);
    return mfma * wgs / 2000.0 / 0.7;
}

// A product of rows and weights, split over k where its tiles are few; `parts` null: not split.
bool product_is_big(long long rows, int n, int dtype) {
    return dtype != SR355_DTYPE_F32 &&
           tiles_are_big(tok_cdiv(rows, Tile256::BM) * tok_cdiv(n, Tile256::BN), SmallShape(dtype).tiles(rows, n));
}
Splits product_splits(long long rows, int n, int k, int sections, int dtype) {
    if (product_is_big(rows, n, dtype)) return {1, 0};
    const SmallShape small(dtype);
    const long long stages = tok_cdiv(k, small.kb / (long long)tok_type_bytes(dtype)) * sections;
    return pick_splits(small.tiles(rows, n), small.slots, stages, (double)rows * n,
                       dtype == SR355_DTYPE_F32 ? stage_us<TileF32>(dtype) : stage_us<Tile128>(dtype));
}

template <typename T>
int reduce_launch(const ReduceArgs &r, int n_jobs, const char *what, hipStream_t stream) {
    long long most = 0;
    for (int i = 0; i < n_jobs; ++i) {
        const long long n = r.job[i].rows * round_up(r.job[i].cols, 8);
        if (n > most) most = n;
    }
    const long long wgs = tok_cdiv(most, 1024);
    hipLaunchKernelGGL((reduce_splits_kernel<T>), dim3((unsigned)(wgs > 2048 ? 2048 : wgs), n_jobs), dim3(256), 0, stream, r);
    return check_hip(hipGetLastError(), what);
}

template <typename T, bool B_RC>
int product_launch(TokGemmArgs &g, const Splits &split, float *parts, const char *what, hipStream_t stream) {
    if (!parts) return gemm_pick<T, false, B_RC, TOK_EPI_STORE>(g, what, stream);
    TokJob &j = g.job[0];
    g.splits = split.n, g.split_stages = split.stages;
    j.part = parts;
    set_tiles<TileSmall<T>>(g, false);
    const int rc = gemm_launch<T, TileSmall<T>, false, B_RC, TOK_EPI_PART>(g, what, stream);
    if (rc != SR355_OK) return rc;
    ReduceArgs r = {};
    r.job[0] = {parts, j.c, j.M, j.N}, r.splits = split.n, r.bias = j.bias;
    return reduce_launch<T>(r, 1, what, stream);
}

// ---- the plan of a call: what is copied, where things lie in the workspace --------------------------------------------
// The row stride, in elements, of a buffer of this file's own: wide rows begin with a line of memory, or a stage's share of a
// row is in two (fp16, 5003 x 501 x 1333, strides 512 and 1344 against 504 and 1336: down 21 against 26 us, gate / up 35
// against 39).
long long row_ld(int cols, int dtype) {
    const int line = 128 / (int)tok_type_bytes(dtype);
    return round_up(cols, cols >= 4 * line ? line : 8);
}
struct Operand {
    const void *p;
    long long ld;     // elements
};
struct Plan {
    size_t at = 0;
    unsigned char *base = nullptr;
    PadArgs pads;
    int n_pads = 0;

    void *take(size_t bytes) {
        void *r = base ? base + at : nullptr;
        at += (bytes + 255) & ~(size_t)255;
        return r;
    }
    // whether 16-byte reads can have the operand as it is
    static bool in_place(const void *p, int cols, long long ld, int dtype) {
        const int e = dtype == SR355_DTYPE_F32 ? 4 : 8;
        return cols % e == 0 && ld % e == 0 && tok_aligned16(p) && ld * (long long)tok_type_bytes(dtype) < (1LL << 22);
    }
    Operand copy(const void *p, long long rows, int cols, long long ld, int dtype) {
        const long long dst_ld = row_ld(cols, dtype);
        void *dst = take((size_t)rows * dst_ld * tok_type_bytes(dtype));
        pads.job[n_pads++] = {p, dst, rows, ld, dst_ld, cols};
        return {dst, dst_ld};
    }
    // the operand as it is where that can be, else its padded copy
    Operand operand(const void *p, long long rows, int cols, long long ld, int dtype) {
        return in_place(p, cols, ld, dtype) ? Operand{p, ld} : copy(p, rows, cols, ld, dtype);
    }
    // The gate and up weights, which the kernels read with one row stride: both as they are, or copies of both (a copy's rows
    // may be longer than the weight's, see row_ld).
    void gate_and_up(const sr355_ffn_args *a, Operand &wg, Operand &wu) {
        const int c = a->channels;
        if (in_place(a->w_gate_dev, c, c, a->dtype) && in_place(a->w_up_dev, c, c, a->dtype)) {
            wg = {a->w_gate_dev, c}, wu = {a->w_up_dev, c};
        } else {
            wg = copy(a->w_gate_dev, a->hidden, c, c, a->dtype);
            wu = copy(a->w_up_dev, a->hidden, c, c, a->dtype);
        }
    }
};

template <typename T>
int run_pads(const Plan &plan, hipStream_t stream) {
    if (!plan.n_pads) return SR355_OK;
    long long most = 0;
    for (int i = 0; i < plan.n_pads; ++i) {
        const long long n = plan.pads.job[i].rows * tok_cdiv(plan.pads.job[i].dst_ld, 512);
        if (n > most) most = n;
    }
    if (most == 0) return SR355_OK;
    const long long wgs = tok_cdiv(most, 4);
    hipLaunchKernelGGL((pad_rows_kernel<T>), dim3((unsigned)(wgs > 4096 ? 4096 : wgs), plan.n_pads), dim3(256), 0, stream, plan.pads);
    return check_hip(hipGetLastError(), "gated_ffn row padding launch");
}

// Rows of h, the kept factors, dg and du: whole groups of eight channels, what a lane of the epilogue stores (zeros behind the
// last channel); wide ones begin with a line of memory.
long long hidden_cols(const sr355_ffn_args *a) { return round_up(a->hidden, 8); }
long long hidden_ld(const sr355_ffn_args *a) { return row_ld(a->hidden, a->dtype); }

size_t hidden_bytes(const sr355_ffn_args *a) {
    return ((size_t)a->rows * hidden_ld(a) * tok_type_bytes(a->dtype) + 255) & ~(size_t)255;
}

// The one-launch kernel of token_narrow.h: 16-bit types, up to 128 channels, nothing kept, and rows for half of the CUs at least
// (a workgroup walks all hidden channels by itself).
bool narrow_fits(const sr355_ffn_args *a) {
    return !a->saved_dev && a->dtype != SR355_DTYPE_F32 && a->channels <= 128 && a->rows >= 64LL * N_CU;
}

// Few rows, the kernels of token_rows.h: reading the weights bounds them.  Their workgroups each read all rows, 16 or fewer
// channels' worth, so with many rows and channels the tiles of 128 rows are faster, split over k for down (bf16, us:
//     rows                 16        32        64
//     gate / up 1024 x 4096    6 / 15    7 / 15   11 / 15
//               2048 x 8192   15 / 22   18 / 22   27 / 22
//     down      1024 x 4096    8 / 10   12 / 10   19 / 12
//               2048 x 8192   14 / 15   22 / 15   37 / 17, rows / tiles).  fp32 tiles are bound by the matrix pipes even then.
constexpr int FEW_ROWS = 64;
bool few_glu(const sr355_ffn_args *a) {
    return a->rows <= 32 || (a->rows <= FEW_ROWS && (a->dtype == SR355_DTYPE_F32 || (long long)a->channels * a->hidden <= (1 << 23)));
}
bool few_down(const sr355_ffn_args *a) {
    return a->rows <= 16 || (a->rows <= FEW_ROWS && (a->dtype == SR355_DTYPE_F32 || (long long)a->channels * a->hidden <= (1 << 21)));
}

// Small blocks of the 16-bit types, whose launches are their starts: h is held in two parts, so that y is rounded once.  The second
// part takes 0.1 to 0.4 us there (16 x 64 x 256: down 3.3 against 3.0 us; 16 x 256 x 1024, beyond: 5.5 against 4.5); larger calls
// would pay half of the down product again.  So a row's y may differ by a step between calls of different sizes.
bool low_kept(const sr355_ffn_args *a) {
    return a->rows <= FEW_ROWS && a->dtype != SR355_DTYPE_F32 && a->rows * a->channels * a->hidden <= (1 << 19);
}

// a call's saved buffer: h, the two kept arrays, their low parts
struct Saved {
    TokKept kept = {};
    void *h = nullptr;
    size_t bytes = 0;
    Saved(const sr355_ffn_args *a, unsigned char *base) {
        auto take = [&](size_t n) {
            void *r = base ? base + bytes : nullptr;
            bytes += (n + 255) & ~(size_t)255;
            return r;
        };
        h = take(hidden_bytes(a)), kept.a = take(hidden_bytes(a)), kept.d = take(hidden_bytes(a));
        if (a->dtype == SR355_DTYPE_F32) return;
        kept.a_low = (unsigned char *)take((size_t)a->rows * hidden_ld(a)), kept.d_low = (unsigned char *)take((size_t)a->rows * hidden_ld(a));
    }
};

struct ForwardPlan : Plan {
    Operand x, wg, wu, wd;
    TokKept kept = {};
    void *h = nullptr, *h_low = nullptr;
    Operand bg = {nullptr, 0}, bu = {nullptr, 0};
    Splits down;
    float *parts = nullptr;

    ForwardPlan(const sr355_ffn_args *a, unsigned char *ws) {
        base = ws;
        x = operand(a->x_dev, a->rows, a->channels, a->x_ld, a->dtype);
        gate_and_up(a, wg, wu);
        wd = operand(a->w_down_dev, a->channels, a->hidden, a->hidden, a->dtype);
        if (a->saved_dev) {
            const Saved s(a, (unsigned char *)a->saved_dev);
            kept = s.kept, h = s.h;
        }
        if (narrow_fits(a)) {
            if (a->b_gate_dev) bg = operand(a->b_gate_dev, 1, a->hidden, hidden_cols(a), a->dtype);
            if (a->b_up_dev) bu = operand(a->b_up_dev, 1, a->hidden, hidden_cols(a), a->dtype);
            return;
        }
        if (!h) h = take(hidden_bytes(a));
        if (few_down(a) && low_kept(a)) h_low = take(hidden_bytes(a));
        if (!few_down(a)) {
            down = product_splits(a->rows, a->channels, a->hidden, 1, a->dtype);
            if (down.n > 1) parts = (float *)take((size_t)down.n * a->rows * round_up(a->channels, 8) * sizeof(float));
            split = down.n > 1;
        }
    }
    bool split = false;
};

// The weight gradients, and with w_down's its bias gradient as the left operand's sums: k is the rows.  Without w_down's, the
// bias gradient takes a product with one column that is not stored.
struct WgradShape {
    bool big;
    Splits split;
};
template <typename G>
long long wgrad_tiles(const sr355_ffn_args *a) {
    auto tiles = [](int M, int N, const void *w, const void *b) { return w || b ? tok_cdiv(M, G::BM) * tok_cdiv(w ? N : 1, G::BN) : 0; };
    return tiles(a->hidden, a->channels, a->dw_gate_dev, nullptr) + tiles(a->hidden, a->channels, a->dw_up_dev, nullptr) +
           tiles(a->channels, a->hidden, a->dw_down_dev, a->db_down_dev);
}
template <typename G>
Splits wgrad_splits(const sr355_ffn_args *a, int slots) {
    const int mats = (a->dw_gate_dev != nullptr) + (a->dw_up_dev != nullptr) + (a->dw_down_dev != nullptr);
    return pick_splits(wgrad_tiles<G>(a), slots, tok_cdiv(a->rows, G::KB / (long long)tok_type_bytes(a->dtype)),
                       (double)mats * a->hidden * a->channels, stage_us<G>(a->dtype));
}
WgradShape wgrad_shape(const sr355_ffn_args *a) {
    if (a->dtype == SR355_DTYPE_F32) return {false, wgrad_splits<TileF32>(a, SmallShape(a->dtype).slots)};
    if (wgrad_tiles<TileWgrad>(a) >= N_CU / 4) return {true, wgrad_splits<TileWgrad>(a, N_CU)};
    return {false, wgrad_splits<Tile128>(a, SmallShape(a->dtype).slots)};
}

// waves of a tile's rows, each of which leaves column sums of dg and du (of at most as many tiles as small ones are)
int sum_rows(const sr355_ffn_args *a) { return a->dtype == SR355_DTYPE_F32 ? TileF32::WM : Tile128::WM; }
static_assert(Tile256::WM == Tile128::WM, "sum_rows");

struct BackwardPlan : Plan {
    Operand x, dy, wg, wu, wd;
    void *dg, *du;
    TokKept kept;
    const void *h;
    float *parts, *row_parts, *dx_parts, *sums;
    WgradShape wgrad;
    Splits dx;
    bool need_hidden;

    BackwardPlan(const sr355_ffn_args *a, unsigned char *ws) {
        base = ws;
        const bool gate_up = a->dw_gate_dev || a->dw_up_dev || a->db_gate_dev || a->db_up_dev;
        need_hidden = a->dx_dev || gate_up;
        x = wg = wu = wd = {nullptr, 0};
        dy = operand(a->dy_dev, a->rows, a->channels, a->dy_ld, a->dtype);
        if (gate_up) x = operand(a->x_dev, a->rows, a->channels, a->x_ld, a->dtype);
        if (a->dx_dev) gate_and_up(a, wg, wu);
        if (need_hidden) wd = operand(a->w_down_dev, a->channels, a->hidden, a->hidden, a->dtype);
        const Saved s(a, (unsigned char *)a->saved_dev);
        kept = s.kept, h = s.h;
        dg = need_hidden ? take(hidden_bytes(a)) : nullptr;
        du = need_hidden ? take(hidden_bytes(a)) : nullptr;
        wgrad = wgrad_shape(a);
        const size_t wide = (size_t)a->hidden * round_up(a->channels, 8), tall = (size_t)a->channels * round_up(a->hidden, 8);
        const size_t weights = (a->dw_gate_dev ? wide : 0) + (a->dw_up_dev ? wide : 0) + (a->dw_down_dev ? tall : 0);
        parts = weights && wgrad.split.n > 1 ? (float *)take(wgrad.split.n * weights * sizeof(float)) : nullptr;
        dx = {1, 0};
        if (a->dx_dev && a->rows > 0) dx = product_splits(a->rows, a->channels, a->hidden, 2, a->dtype);
        dx_parts = dx.n > 1 ? (float *)take((size_t)dx.n * a->rows * round_up(a->channels, 8) * sizeof(float)) : nullptr;
        row_parts = wgrad.split.n > 1 && a->db_down_dev ? (float *)take((size_t)wgrad.split.n * round_up(a->channels, 8) * sizeof(float)) : nullptr;
        sums = a->db_gate_dev || a->db_up_dev
                   ? (float *)take((size_t)tok_cdiv(a->rows, SmallShape(a->dtype).bm) * sum_rows(a) * 2 * hidden_cols(a) * sizeof(float)) : nullptr;
    }
};

bool ffn_args_ok(const char *who, const sr355_ffn_args *a, bool backward) {
    if (!a || !tok_dtype_ok(a->dtype) || a->activation < 0 || a->activation > SR355_ACT_SIGMOID || a->rows < 0 ||
        a->rows > 0x7fffff00LL || a->channels < 1 || a->hidden < 1 || a->channels > (1 << 20) || a->hidden > (1 << 20) ||
        a->x_ld < a->channels || (backward && a->dy_ld < a->channels)) {
        if (!a) set_error("%s: null arguments", who);
        else
            set_error("%s: bad arguments (dtype=%d activation=%d rows=%lld channels=%d hidden=%d, row strides %lld and %lld; "
                      "widths up to 2^20, fewer than 2^31 rows)", who, a->dtype, a->activation, a->rows, a->channels, a->hidden,
                      a->x_ld, a->dy_ld);
        return false;
    }
    return true;
}

template <typename T, int TG, bool GLU, int WAVES, bool LOW>
int few_rows(TokRowsArgs a, const char *what, hipStream_t stream) {
    a.channels = 16;
    while (a.channels > 4 && tok_cdiv(a.n_store, a.channels) < N_CU) a.channels /= 2;
    hipLaunchKernelGGL((tok_rows_kernel<T, TG, GLU, WAVES, LOW>), dim3((unsigned)tok_cdiv(a.n_store, a.channels)), dim3(64 * WAVES), 0, stream, a);
    return check_hip(hipGetLastError(), what);
}
template <typename T, bool GLU, bool LOW = false>
int few_rows_any(const TokRowsArgs &a, const char *what, hipStream_t stream) {
    if (a.rows <= 16) return few_rows<T, 1, GLU, GLU ? 8 : 16, LOW>(a, what, stream);
    if (a.rows <= 32) return few_rows<T, 2, GLU, GLU ? 8 : 16, LOW>(a, what, stream);
    return few_rows<T, 4, GLU, GLU ? 4 : 8, LOW>(a, what, stream);
}

template <typename T>
int ffn_glu_few(const sr355_ffn_args *a, const ForwardPlan &p, hipStream_t stream) {
    TokRowsArgs g = {};
    g.x = (const unsigned char *)p.x.p, g.x_ld = p.x.ld * sizeof(T);
    g.w = (const unsigned char *)p.wg.p, g.w2 = (const unsigned char *)p.wu.p, g.w_ld = p.wg.ld * sizeof(T);
    g.rows = (int)a->rows, g.N = a->hidden, g.k_bytes = (int)(a->channels * sizeof(T));
    g.bias = a->b_gate_dev, g.bias2 = a->b_up_dev, g.act = a->activation;
    g.out = p.h, g.out_low = p.h_low, g.kept = p.kept, g.out_ld = hidden_ld(a), g.n_store = (int)hidden_cols(a);
    return few_rows_any<T, true>(g, "gated_ffn gate / up launch", stream);
}
template <typename T>
int ffn_down_few(const sr355_ffn_args *a, const ForwardPlan &p, hipStream_t stream) {
    TokRowsArgs d = {};
    d.x = (const unsigned char *)p.h, d.x_low = (const unsigned char *)p.h_low, d.x_ld = hidden_ld(a) * sizeof(T);
    d.w = (const unsigned char *)p.wd.p, d.w_ld = p.wd.ld * sizeof(T);
    d.rows = (int)a->rows, d.N = a->channels, d.k_bytes = (int)(a->hidden * sizeof(T)), d.bias = a->b_down_dev;
    d.out = a->y_dev, d.out_ld = a->channels, d.n_store = a->channels;
    if constexpr (sizeof(T) == 2) {
        if (p.h_low) return few_rows_any<T, false, true>(d, "gated_ffn down launch", stream);
    }
    return few_rows_any<T, false>(d, "gated_ffn down launch", stream);
}

template <typename T, int CP, int KIND>
void narrow_launch_width(const TokNarrowArgs &n, hipStream_t stream) {
    const dim3 grid((unsigned)tok_cdiv(n.rows, TokNarrow<CP>::ROWS));
    if (n.bg || n.bu) hipLaunchKernelGGL((tok_narrow_kernel<T, CP, KIND, true>), grid, dim3(256), 0, stream, n);
    else hipLaunchKernelGGL((tok_narrow_kernel<T, CP, KIND, false>), grid, dim3(256), 0, stream, n);
}
template <typename T, int KIND>
void narrow_launch(const TokNarrowArgs &n, hipStream_t stream) {
    if (n.C <= 64) narrow_launch_width<T, 64, KIND>(n, stream);
    else narrow_launch_width<T, 128, KIND>(n, stream);
}

template <typename T>
int ffn_forward_narrow(const sr355_ffn_args *a, const ForwardPlan &p, hipStream_t stream) {
    TokNarrowArgs n = {};
    n.x = (const unsigned char *)p.x.p, n.x_ld = p.x.ld * sizeof(T);
    n.wg = (const unsigned char *)p.wg.p, n.wu = (const unsigned char *)p.wu.p, n.w_ld = p.wg.ld * sizeof(T);
    n.wd = (const unsigned char *)p.wd.p, n.wd_ld = p.wd.ld * sizeof(T);
    n.bg = (const unsigned char *)p.bg.p, n.bu = (const unsigned char *)p.bu.p, n.bd = a->b_down_dev;
    n.y = a->y_dev, n.y_ld = a->channels, n.rows = a->rows, n.C = a->channels, n.F = a->hidden, n.act = a->activation;
    if (a->activation == SR355_ACT_SILU) narrow_launch<T, SR355_ACT_SILU>(n, stream);
    else if (a->activation == SR355_ACT_GELU) narrow_launch<T, SR355_ACT_GELU>(n, stream);
    else if (a->activation == SR355_ACT_RELU) narrow_launch<T, SR355_ACT_RELU>(n, stream);
    else narrow_launch<T, SR355_ACT_SIGMOID>(n, stream);
    return check_hip(hipGetLastError(), "gated_ffn narrow launch");
}

template <typename T>
int ffn_forward(const sr355_ffn_args *a, hipStream_t stream) {
    ForwardPlan p(a, (unsigned char *)a->workspace_dev);
    int rc = run_pads<T>(p, stream);
    if (rc != SR355_OK) return rc;
    if constexpr (sizeof(T) == 2) {
        if (narrow_fits(a)) return ffn_forward_narrow<T>(a, p, stream);
    }
    TokGemmArgs g = {};
    g.n_jobs = 1, g.sections = 1, g.act = a->activation, g.K = a->channels;
    TokJob &j = g.job[0];
    j.a[0] = (const unsigned char *)p.x.p, j.a_ld = p.x.ld * sizeof(T);
    j.b[0] = (const unsigned char *)p.wg.p, j.b[1] = (const unsigned char *)p.wu.p, j.b_ld = p.wg.ld * sizeof(T);
    j.M = (int)a->rows, j.N = a->hidden, j.bias = a->b_gate_dev;
    g.bias_up = a->b_up_dev, g.kept = p.kept, g.h = p.h, g.h_ld = hidden_ld(a);
    rc = few_glu(a) ? ffn_glu_few<T>(a, p, stream) : gemm_pick<T, false, false, TOK_EPI_GLU>(g, "gated_ffn gate / up launch", stream);
    if (rc != SR355_OK) return rc;
    if (few_down(a)) return ffn_down_few<T>(a, p, stream);
    TokGemmArgs d = {};
    d.n_jobs = 1, d.sections = 1, d.K = a->hidden;
    TokJob &k = d.job[0];
    k.a[0] = (const unsigned char *)p.h, k.a_ld = hidden_ld(a) * sizeof(T);
    k.b[0] = (const unsigned char *)p.wd.p, k.b_ld = p.wd.ld * sizeof(T);
    k.M = (int)a->rows, k.N = a->channels, k.bias = a->b_down_dev, k.c = a->y_dev, k.c_ld = a->channels;
    return product_launch<T, false>(d, p.down, p.split ? p.parts : nullptr, "gated_ffn down launch", stream);
}

template <typename T, typename G, bool SUMS>
int wgrad_launch(TokGemmArgs &g, bool part, hipStream_t stream) {
    set_tiles<G>(g, false);
    return part ? gemm_launch<T, G, true, true, TOK_EPI_PART, SUMS>(g, "gated_ffn weight gradient launch", stream)
                : gemm_launch<T, G, true, true, TOK_EPI_STORE, SUMS>(g, "gated_ffn weight gradient launch", stream);
}

template <typename T>
int ffn_wgrad(const sr355_ffn_args *a, const BackwardPlan &p, hipStream_t stream) {
    TokGemmArgs g = {};
    g.sections = 1, g.K = (int)a->rows, g.splits = p.wgrad.split.n, g.split_stages = p.wgrad.split.stages;
    ReduceArgs r = {};
    float *parts = p.parts, *row_parts = p.row_parts;
    int n_out = 0;
    auto add = [&](const void *l, long long l_ld, const void *q, long long q_ld, int M, int N, void *out, void *sums) {
        if (!out && !sums) return;
        TokJob &j = g.job[g.n_jobs++];
        j.a[0] = (const unsigned char *)l, j.a_ld = l_ld * sizeof(T);
        j.b[0] = (const unsigned char *)q, j.b_ld = q_ld * sizeof(T);
        j.M = M, j.N = out ? N : 1, j.c = out, j.c_ld = N, j.row_sums = sums;
        if (g.splits == 1) return;
        if (out) {
            j.part = parts, parts += (size_t)g.splits * M * round_up(N, 8);
            r.job[n_out++] = {j.part, out, M, N};
        }
        if (sums) {
            j.row_part = row_parts, row_parts += (size_t)g.splits * round_up(M, 8);
            r.job[n_out++] = {j.row_part, sums, 1, M};
        }
    };
    add(p.dg, hidden_ld(a), p.x.p, p.x.ld, a->hidden, a->channels, a->dw_gate_dev, nullptr);
    add(p.du, hidden_ld(a), p.x.p, p.x.ld, a->hidden, a->channels, a->dw_up_dev, nullptr);
    add(p.dy.p, p.dy.ld, p.h, hidden_ld(a), a->channels, a->hidden, a->dw_down_dev, a->db_down_dev);
    if (!g.n_jobs) return SR355_OK;
    const bool part = g.splits > 1;
    const bool sums = a->db_down_dev != nullptr;
    int rc;
    if constexpr (sizeof(T) == 2) {
        if (p.wgrad.big) rc = sums ? wgrad_launch<T, TileWgrad, true>(g, part, stream) : wgrad_launch<T, TileWgrad, false>(g, part, stream);
        else rc = sums ? wgrad_launch<T, Tile128, true>(g, part, stream) : wgrad_launch<T, Tile128, false>(g, part, stream);
    } else {
        rc = sums ? wgrad_launch<T, TileF32, true>(g, part, stream) : wgrad_launch<T, TileF32, false>(g, part, stream);
    }
    if (rc != SR355_OK || !part) return rc;
    r.splits = p.wgrad.split.n;
    return reduce_launch<T>(r, n_out, "gated_ffn weight gradient reduction launch", stream);
}

template <typename T>
int ffn_backward(const sr355_ffn_args *a, hipStream_t stream) {
    BackwardPlan p(a, (unsigned char *)a->workspace_dev);
    int rc = run_pads<T>(p, stream);
    if (rc != SR355_OK) return rc;
    int n_sums = 0;
    if (p.need_hidden && a->rows > 0) {
        TokGemmArgs g = {};
        g.n_jobs = 1, g.sections = 1, g.act = a->activation, g.K = a->channels;
        TokJob &j = g.job[0];
        j.a[0] = (const unsigned char *)p.dy.p, j.a_ld = p.dy.ld * sizeof(T);
        j.b[0] = (const unsigned char *)p.wd.p, j.b_ld = p.wd.ld * sizeof(T);
        j.M = (int)a->rows, j.N = a->hidden;
        g.g = p.dg, g.u = p.du, g.kept = p.kept, g.h_ld = hidden_ld(a);
        g.sums = p.sums;
        rc = p.sums ? gemm_pick<T, false, true, TOK_EPI_GLU_GRAD, true>(g, "gated_ffn hidden gradient launch", stream)
                    : gemm_pick<T, false, true, TOK_EPI_GLU_GRAD>(g, "gated_ffn hidden gradient launch", stream);
        if (rc != SR355_OK) return rc;
        n_sums = j.tiles_m * sum_rows(a);
    }
    if (p.sums) {
        const long long first[2] = {0, hidden_cols(a)};
        const int count[2] = {a->hidden, a->hidden};
        void *const out[2] = {a->db_gate_dev, a->db_up_dev};
        rc = launch_tok_sum_parts(p.sums, n_sums, 2 * hidden_cols(a), first, count, out, 2, a->dtype, stream);
        if (rc != SR355_OK) return rc;
    }
    if (a->dx_dev && a->rows > 0) {
        TokGemmArgs g = {};
        g.n_jobs = 1, g.sections = 2, g.K = a->hidden;
        TokJob &j = g.job[0];
        j.a[0] = (const unsigned char *)p.dg, j.a[1] = (const unsigned char *)p.du, j.a_ld = hidden_ld(a) * sizeof(T);
        j.b[0] = (const unsigned char *)p.wg.p, j.b[1] = (const unsigned char *)p.wu.p, j.b_ld = p.wg.ld * sizeof(T);
        j.M = (int)a->rows, j.N = a->channels, j.c = a->dx_dev, j.c_ld = a->channels;
        rc = product_launch<T, true>(g, p.dx, p.dx_parts, "gated_ffn data gradient launch", stream);
        if (rc != SR355_OK) return rc;
    }
    return ffn_wgrad<T>(a, p, stream);
}
}  // namespace

}  // namespace sr355

using namespace sr355;

extern "C" {

size_t sr355_gated_ffn_saved_bytes(const sr355_ffn_args *a) {
    if (!ffn_args_ok("gated_ffn_saved_bytes", a, false)) return 0;
    return Saved(a, nullptr).bytes + 256;
}

size_t sr355_gated_ffn_workspace_bytes(const sr355_ffn_args *a, int backward) {
    if (!ffn_args_ok("gated_ffn_workspace_bytes", a, backward != 0)) return 0;
    return (backward ? BackwardPlan(a, nullptr).at : ForwardPlan(a, nullptr).at) + 256;
}

int sr355_gated_ffn_fwd(const sr355_ffn_args *a, void *stream) {
    if (!ffn_args_ok("gated_ffn_fwd", a, false)) return SR355_ERR_INVALID;
    if (a->rows == 0) return SR355_OK;
    const size_t need = sr355_gated_ffn_workspace_bytes(a, 0);
    if (!a->x_dev || !a->w_gate_dev || !a->w_up_dev || !a->w_down_dev || !a->y_dev || !a->workspace_dev ||
        !tok_aligned16(a->workspace_dev) || a->workspace_bytes < need || !tok_aligned16(a->saved_dev) ||
        (a->saved_dev && a->saved_bytes < sr355_gated_ffn_saved_bytes(a))) {
        set_error("gated_ffn_fwd: null tensor, or workspace / saved buffer not 16-byte aligned or smaller than %zu / %zu bytes", need,
                  sr355_gated_ffn_saved_bytes(a));
        return SR355_ERR_INVALID;
    }
    if (a->dtype == SR355_DTYPE_F32) return ffn_forward<float>(a, (hipStream_t)stream);
    if (a->dtype == SR355_DTYPE_BF16) return ffn_forward<bf16_t>(a, (hipStream_t)stream);
    return ffn_forward<f16_t>(a, (hipStream_t)stream);
}

int sr355_gated_ffn_bwd(const sr355_ffn_args *a, void *stream) {
    if (!ffn_args_ok("gated_ffn_bwd", a, true)) return SR355_ERR_INVALID;
    const size_t need = sr355_gated_ffn_workspace_bytes(a, 1);
    if ((a->rows > 0 && (!a->x_dev || !a->dy_dev || !a->saved_dev || a->saved_bytes < sr355_gated_ffn_saved_bytes(a))) ||
        !tok_aligned16(a->saved_dev) || !a->w_gate_dev || !a->w_up_dev || !a->w_down_dev || !a->workspace_dev ||
        !tok_aligned16(a->workspace_dev) || a->workspace_bytes < need) {
        set_error("gated_ffn_bwd: null tensor, or workspace / saved buffer not 16-byte aligned or smaller than %zu / %zu bytes", need,
                  sr355_gated_ffn_saved_bytes(a));
        return SR355_ERR_INVALID;
    }
    if (a->dtype == SR355_DTYPE_F32) return ffn_backward<float>(a, (hipStream_t)stream);
    if (a->dtype == SR355_DTYPE_BF16) return ffn_backward<bf16_t>(a, (hipStream_t)stream);
    return ffn_backward<f16_t>(a, (hipStream_t)stream);
}

}  // extern "C"
