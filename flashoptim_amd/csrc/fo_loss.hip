// Cross entropy over a vocabulary straight from hidden states, without the logits in memory, and its gradients.
//
//   z = x W'      lse[i] = log sum_v exp(z[i][v])      loss[i] = lse[i] - (1 - e) z[i][t_i] - e mean_v z[i][v]      (0 for ignored targets)
//   G[i][v] = f_i (exp(z[i][v] - lse[i]) - e / V - (1 - e) [v = t_i])        dx = G W        dW = G' x
//
// with f_i what the loss of row i is multiplied by on its way back, over the number of targets where the loss is a mean.
//
// Forward: a tile of z stays in a workgroup's accumulators; out go each row's maximum, its sum of exponentials relative to that, and the
// target's logit where the tile holds it: 8 bytes for a row of a wavefront's part of the tile.  Another launch joins the parts.
// Backward: a piece of the vocabulary at a time.  The piece's logits are computed again (a product more, and nothing of tokens x vocabulary size kept
// from the forward pass), turned into G in the same accumulators and written, 16 bits a value; then one product adds
// G's share to dx (fp32 sums between pieces), another makes the piece's rows of dW, complete.
//
// Types.  bf16 and fp16 operands go into the matrix cores as they are, sums are fp32.  G is rounded to the operands' type once, as the
// other operand of its products is; the factors f_i are first divided by the largest of them (and multiplied by 2^15 for fp16, so that probabilities down to 2^-39
// survive), which the products' results are multiplied by at the end: where all are equal, as in a mean, they are 1, and the entry p - 1 of an unlikely
// target rounds to almost itself.  What the target's entry, by far the largest of most rows, loses in its rounding goes into dx all the same: that times the
// target's row of W is added in fp32, which reads a row of W beside every row of dx (of a backward pass of 4096 x 4096 over 1024 6 us in 164, of 4096 x 512 over 64 1 in 29, of
// 8192 x 4096 over 128256 less than is measured).  dW has the entries as they were rounded.  fp32 operands go into the fp32 instructions, a sixteenth of the rate; or, where the work is large enough to pay for laying
// them out (in_parts), they are cut into three bf16 parts of 8 bits each, a = a1 + a2 + a3
// exactly, and the six products a3 b1, a2 b2, a1 b3, a2 b1, a1 b2, a1 b1 are one contraction over six times the length: what is left
// out is below 2^-23 of a product.  The small ones come first, so that the sums are small while most of the additions round.
//
// Operands are read in place where their rows are whole 16-byte pieces, aligned; others are laid out first.  The contracted axis is filled up to half a stage with zeros on
// one side of a product.  G = f (p - ...) is written once, by rows, and read by rows for dx and by columns for dW, W by rows for the logits and by columns for dx: the product core reads
// either way.  Rows of ignored targets are left out of dW by zeros on both sides, so that what stands in them (infinities, NaN) does not matter: x is copied for that.
#include "fo_gemm.h"
#include "fo_host.h"

namespace fo {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kMinusInf = -__builtin_inff();
constexpr int kIgnored = -1, kNone = -2;    // labels

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// ------------------------------------------------------------------------------------------- operands
// Eight neighbouring values of a row as a product's operands have them: rounded to a 16-bit type, as they are, or the three parts of each, `part_stride` bytes apart.
// Returned is what was lost of v[at] by that (0 where at is none of them).
template <int DT, class Product> struct OperandOf {
    static constexpr int kBytes = 2;
    __device__ __forceinline__ static float store(const float (&v)[8], char* p, int64_t, int at) {
        Pack<2, 8> d;
        float lost = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
            float a, b;
            narrow_pair<DT, 8>(d, k, v[k], v[k + 1], a, b);
            if (at == k) lost = v[k] - a;
            if (at == k + 1) lost = v[k + 1] - b;
        }
        store_piece<2, 8>(d, p, 8);
        return lost;
    }
};
template <> struct OperandOf<DT_F32, F32Product> {
    static constexpr int kBytes = 4;
    __device__ __forceinline__ static float store(const float (&v)[8], char* p, int64_t, int) {
        store_values<DT_F32>(v, p, 8);
        return 0.0f;
    }
};
template <> struct OperandOf<DT_F32, Bf16PartsProduct> {
    static constexpr int kBytes = 2;
    __device__ __forceinline__ static float store(const float (&v)[8], char* p, int64_t part_stride, int) {
        u32x4 part[3];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            u32 lo[3], hi[3];
            cut(v[2 * k], lo);
            cut(v[2 * k + 1], hi);
#pragma unroll
            for (int i = 0; i < 3; ++i) part[i][k] = __builtin_amdgcn_perm(hi[i], lo[i], 0x07060302u);
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) *reinterpret_cast<FO_GLOBAL u32x4*>((FO_GLOBAL char*)p + i * part_stride) = part[i];
        return 0.0f;
    }
    // Eight bits of the significand at a time, cut off: nothing overflows, and the rest is exact.
    __device__ __forceinline__ static void cut(float x, u32 (&part)[3]) {
        part[0] = as_u32(x) & 0xffff0000u;
        const bool finite = (as_u32(x) & 0x7f800000u) != 0x7f800000u;
        if (!finite && x != x) part[0] |= 0x00400000u;
        const float rest = finite ? x - as_f32(part[0]) : 0.0f;
        part[1] = as_u32(rest) & 0xffff0000u;
        part[2] = as_u32(rest - as_f32(part[1])) & 0xffff0000u;
    }
};
// Which part each segment of a product in parts takes, of its left and of its right operand: 2 1 0 1 0 0 and 0 1 2 0 1 0, the first in the low bits.
constexpr u32 kLeftOrder = 2u | 1u << 2 | 0u << 4 | 1u << 6, kRightOrder = 0u | 1u << 2 | 2u << 4 | 0u << 6 | 1u << 8;

struct FormArgs {
    const char* x;
    char* out;
    const int* labels;        // rows of x whose label is kIgnored count as zeros; or null
    int64_t stride;           // of x, in values
    int64_t part_stride;      // of out, in bytes
    int rows, cols;           // of x
    int out_rows, length;     // of out: filled up with zeros
};
// Rows as operand rows, eight values a thread.  Bound by memory: 8192 x 4096 bf16 in 22 us (6.0 TB/s).
template <int DT, class Product> __global__ __launch_bounds__(256) void form_kernel(FormArgs a) {
    typedef OperandOf<DT, Product> To;
    const int pieces = a.length / 8;
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x, r = k / pieces;
    const int c = (int)(k - r * pieces) * 8;
    if (r >= a.out_rows) return;
    float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (r < a.rows && c < a.cols && !(a.labels && a.labels[r] == kIgnored)) load_values<DT>(v, a.x + (r * a.stride + c) * DTypeInfo<DT>::bytes, a.cols - c);
    To::store(v, a.out + (r * a.length + c) * To::kBytes, a.part_stride, -1);
}

// ------------------------------------------------------------------------------------------- forward
struct Targets {
    const void* p;
    int bytes;
    __device__ __forceinline__ int64_t operator[](int64_t i) const {
        return bytes == 8 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
    }
};

template <int CTRL> __device__ __forceinline__ float of_lane(float x) {
    return as_f32((u32)__builtin_amdgcn_mov_dpp((int)as_u32(x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float max_of_16(float x) {
    x = fmaxf(x, of_lane<0xb1>(x));
    x = fmaxf(x, of_lane<0x4e>(x));
    x = fmaxf(x, of_lane<0x141>(x));
    return fmaxf(x, of_lane<0x140>(x));
}
__device__ __forceinline__ float sum_of_16(float x) {
    x += of_lane<0xb1>(x);
    x += of_lane<0x4e>(x);
    x += of_lane<0x141>(x);
    return x + of_lane<0x140>(x);
}

struct LogitsArgs {
    Operand x, weight;
    int row_bytes, segment_stages;
    Targets targets;    // of row `first` on
    int64_t first;
    f32x2* stats;       // [part][row]: maximum, and sum of exponentials relative to it
    float* sums;        // [part][row]: sum of logits, or null
    float* picked;      // the target's logit
};

// What a grid of result tiles does first: which one is mine.
template <class Tile> __device__ __forceinline__ bool my_tile(int rows, int cols, int& row0, int& col0) {
    const int down = (rows + Tile::kTile - 1) / Tile::kTile, across = (cols + Tile::kTile - 1) / Tile::kTile;
    const int64_t t = tile_of_seat(blockIdx.x & 7, blockIdx.x >> 3, (int64_t)down * across);
    if (t < 0) return false;
    int i, j;
    tile_at((int)t, down, across, i, j);
    row0 = i * Tile::kTile;
    col0 = j * Tile::kTile;
    return true;
}

// A tile of z, then out of the accumulators each row's maximum and sum over a wavefront's WT columns: a lane has four rows of every sixteen and every sixteenth column, so both
// are a few operations in registers and four exchanges between sixteen neighbouring lanes.  Bound by the matrix cores: 8192 x 4096 over 128256 in 6.4 ms, 1350 TFLOP/s (a library
// product of that size, which writes its result, 6.0); 13 of a tile's 101 us are its first loads and this.  With few rows bound by the weight's bytes: 5 rows 163 us, 6.4 TB/s.
template <class Product, int WT, int STAGES> __global__ __launch_bounds__(256, WT >= 96 ? 1 : 2) void logits_kernel(LogitsArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef GemmTile<Product, WT, STAGES> Tile;
    int row0, col0;
    if (!my_tile<Tile>(a.x.rows, a.weight.rows, row0, col0)) return;
    Tile tile(smem);
    tile.segment_stages = a.segment_stages;
    tile.multiply(a.x, a.weight, row0, col0, a.row_bytes);
    const int rows = a.x.rows, cols = a.weight.rows;
    const int r0 = row0 + (tile.wave >> 1) * WT + (tile.lane >> 4) * 4, part0 = col0 + (tile.wave & 1) * WT, mine = tile.lane & 15;
    if (part0 >= cols) return;
    const int64_t part = part0 / WT;
    // which column each row's target is: looked up before anything is stored, or every row waits for its own
    int* wanted = reinterpret_cast<int*>(smem) + tile.wave * WT;
#pragma unroll
    for (int k = tile.lane; k < WT; k += 64) {
        const int r = row0 + (tile.wave >> 1) * WT + k;
        const int64_t at = a.targets[a.first + (r < rows ? r : rows - 1)] - part0;    // one that is ignored, or none, may be found too: nobody asks for it
        wanted[k] = r < rows && at >= 0 && at < WT ? (int)at : -1;
    }
    Tile::same_wave();
#pragma unroll
    for (int i = 0; i < Tile::kFrags; ++i) {
        const i32x4 picks = *reinterpret_cast<const i32x4*>(wanted + i * 16 + (tile.lane >> 4) * 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int r = r0 + i * 16 + k;
            float v[Tile::kFrags], most = kMinusInf;
#pragma unroll
            for (int j = 0; j < Tile::kFrags; ++j) {
                v[j] = part0 + j * 16 + mine < cols ? tile.acc[i][j][k] : kMinusInf;
                most = fmaxf(most, v[j]);
            }
            most = max_of_16(most);
            const float base = most == kMinusInf ? 0.0f : most;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < Tile::kFrags; ++j) sum += exp_of(v[j] - base);
            sum = sum_of_16(sum);
            if (picks[k] >= 0 && (picks[k] & 15) == mine) {
#pragma unroll
                for (int j = 0; j < Tile::kFrags; ++j)
                    if (j == picks[k] >> 4) a.picked[r] = v[j];
            }
            if (mine == 0 && r < rows) a.stats[part * rows + r] = f32x2{most, sum};
            if (a.sums) {
                float all = 0.0f;
#pragma unroll
                for (int j = 0; j < Tile::kFrags; ++j) all += part0 + j * 16 + mine < cols ? v[j] : 0.0f;
                all = sum_of_16(all);
                if (mine == 0 && r < rows) a.sums[part * rows + r] = all;
            }
        }
    }
}

struct JoinArgs {
    const f32x2* stats;
    const float *sums, *picked;
    Targets targets;
    int64_t first, ignore, vocabulary;
    float *most, *log_sum, *loss;    // of each row the largest logit, the log of the sum of exponentials relative to it
    int* labels;
    int rows, parts;
    float smoothing;
};
struct Exps {
    float most, sum;
    __device__ __forceinline__ void add(float m, float s) {
        const float top = fmaxf(most, m), base = top == kMinusInf ? 0.0f : top;
        sum = sum * exp_of(most - base) + s * exp_of(m - base);
        most = top;
    }
};
// Rows' parts joined: ROWS rows a workgroup, each by 1024 / ROWS threads.  Few rows have many parts: five rows of 4008 parts take 44 us with 64 rows to a
// workgroup, 6 with one.
template <int ROWS> __global__ __launch_bounds__(1024) void loss_join_kernel(JoinArgs a) {
    constexpr int kSlices = 1024 / ROWS;
    __shared__ float most[1024], sum[1024], all[1024];
    const int slice = threadIdx.x / ROWS, row = blockIdx.x * ROWS + threadIdx.x % ROWS;
    Exps e{kMinusInf, 0.0f};
    float logits = 0.0f;
    if (row < a.rows) {
#pragma unroll 4
        for (int p = slice; p < a.parts; p += kSlices) {
            const f32x2 v = a.stats[(int64_t)p * a.rows + row];
            e.add(v.x, v.y);
            if (a.sums) logits += a.sums[(int64_t)p * a.rows + row];
        }
    }
#pragma unroll 1
    for (int half = kSlices / 2; half > 0; half >>= 1) {    // the upper half of the slices that are left hands over to the lower
        most[threadIdx.x] = e.most;
        sum[threadIdx.x] = e.sum;
        all[threadIdx.x] = logits;
        __syncthreads();
        if (slice < half) {
            e.add(most[threadIdx.x + half * ROWS], sum[threadIdx.x + half * ROWS]);
            logits += all[threadIdx.x + half * ROWS];
        }
        __syncthreads();
    }
    if (slice != 0 || row >= a.rows) return;
    const float log_sum = __builtin_logf(e.sum);
    const int64_t target = a.targets[a.first + row];
    const int label = target == a.ignore ? kIgnored : target >= 0 && target < a.vocabulary ? (int)target : kNone;
    float loss = 0.0f;
    if (label == kNone) loss = __builtin_nanf("");
    else if (label != kIgnored) {
        // from the maximum, not from lse, whose rounding is as large as the loss of a target that is likely among large logits
        loss = e.most - a.picked[row];
        if (a.smoothing > 0.0f) loss = (1.0f - a.smoothing) * loss + a.smoothing * (e.most - logits / (float)a.vocabulary);
        loss += log_sum;
    }
    a.most[row] = e.most;
    a.log_sum[row] = log_sum;
    a.loss[row] = loss;
    a.labels[row] = label;
}

// The losses' sum, over their number where a mean is wanted; count: that number.
__global__ __launch_bounds__(1024) void loss_reduce_kernel(const float* losses, const int* labels, int64_t n, int reduction, float* loss, float* count) {
    __shared__ double sums[16];
    __shared__ int counts[16];
    double sum = 0.0;
    int kept = 0;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        sum += losses[i];
        kept += labels[i] != kIgnored;
    }
    for (int d = 1; d < 64; d <<= 1) { sum += __shfl_xor(sum, d); kept += __shfl_xor(kept, d); }
    if ((threadIdx.x & 63) == 0) { sums[threadIdx.x >> 6] = sum; counts[threadIdx.x >> 6] = kept; }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int w = 1; w < 16; ++w) { sum += sums[w]; kept += counts[w]; }
    loss[0] = (float)(reduction == FO_REDUCE_MEAN ? sum / (double)kept : sum);
    count[0] = (float)kept;
}

// ------------------------------------------------------------------------------------------- backward
// What the products' results are multiplied by at the end: f_i over the factors that went into G.  The upstream of a sum or a mean is that itself, over the number of
// targets where the loss is a mean; the factors are 1 then, and no launch is needed for them.
struct Scale {
    const float* p;         // the upstream, or what loss_factors_kernel made of many
    const float* count;     // or null
    float over;             // `top`
    bool mean;
    __device__ __forceinline__ float value() const {
        if (!count) return p[0] * over;
        if (count[0] == 0.0f) return 0.0f;    // no targets, no gradients
        return mean ? p[0] * (1.0f / count[0]) * over : p[0] * over;
    }
};

// factors[i]: f_i over the largest magnitude among them, times `top` (a power of two); scale[0]: that magnitude.
__global__ __launch_bounds__(1024) void loss_factors_kernel(const float* upstream, int64_t stride, const int* labels, int64_t n, int reduction, const float* count,
                                                            float top, float* factors, float* scale) {
    __shared__ float mosts[16];
    const float share = reduction == FO_REDUCE_MEAN ? 1.0f / count[0] : 1.0f;
    float most = 0.0f;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        const float f = fabsf(upstream[i * stride] * share);
        if (labels[i] >= 0 && f < __builtin_inff()) most = fmaxf(most, f);
    }
    for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    if ((threadIdx.x & 63) == 0) mosts[threadIdx.x >> 6] = most;
    __syncthreads();
    most = mosts[0];
    for (int w = 1; w < 16; ++w) most = fmaxf(most, mosts[w]);
    if (most == 0.0f) most = 1.0f;
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
        const float f = upstream[i * stride] * share / most * top;
        factors[i] = labels[i] == kIgnored ? 0.0f : labels[i] == kNone ? __builtin_nanf("") : f;
    }
    if (threadIdx.x == 0) scale[0] = most;
}

struct GradArgs {
    Operand x, weight;     // of a piece of the vocabulary
    int row_bytes, segment_stages;
    const int* labels;
    const float *most, *log_sum, *factors;    // no factors: `top` for every row
    float top;
    char* grad;            // G as operand rows over the piece
    float* lost;           // of each row with a target: what its target's entry lost in its rounding; or null
    int64_t part_stride;
    int length;            // of G's rows
    int first;             // the piece's first token of the vocabulary
    float kept, even;      // 1 - e, e / V
};
template <int DT, class Product> struct GradOut {
    static constexpr bool kColumns = false;
    typedef OperandOf<DT, Product> To;
    const GradArgs& a;
    struct In { float most, over, factor; int label; };
    __device__ __forceinline__ void begin(int) const {}
    __device__ __forceinline__ void load(int i, int, In& in) const {
        if (i >= a.x.rows) return;
        in.most = a.most[i];
        in.over = a.log_sum[i] * kLog2e;
        in.label = a.labels[i];
        in.factor = a.factors ? a.factors[i] : in.label == kNone ? __builtin_nanf("") : a.top;
    }
    __device__ __forceinline__ void row(int i, int j, In in, float (&v)[8]) const {
        if (i >= a.x.rows || j >= a.length) return;
        const int at = in.label - a.first - j;    // among the eight, if the target is
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float g = __builtin_amdgcn_exp2f(fmaf(v[k] - in.most, kLog2e, -in.over)) - a.even;    // lse would be rounded to the step of large logits
            if (at == k) g -= a.kept;
            v[k] = in.label == kIgnored || j + k >= a.weight.rows ? 0.0f : g * in.factor;
        }
        const float lost = To::store(v, a.grad + ((int64_t)i * a.length + j) * To::kBytes, a.part_stride, at);
        if (a.lost && at >= 0 && at < 8) a.lost[i] = lost;
    }
};
// The logits again and G of them.  8192 rows, 16128 tokens of a vocabulary: 890 us (1210 TFLOP/s), 50 more than the product alone.
template <int DT, class Product, int WT, int STAGES> __global__ __launch_bounds__(256, WT >= 96 ? 1 : 2) void grad_kernel(GradArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef GemmTile<Product, WT, STAGES> Tile;
    int row0, col0;
    if (!my_tile<Tile>(a.x.rows, a.weight.rows, row0, col0)) return;
    Tile tile(smem);
    tile.segment_stages = a.segment_stages;
    tile.multiply(a.x, a.weight, row0, col0, a.row_bytes);
    GradOut<DT, Product> out{a};
    tile.finish(row0, col0, out);
}

// rows x cols of a product; `parts` of the contraction, part_stages each, may go to workgroups of their own, each with a result of its own in `sums`.
struct GradProductArgs {
    Operand left, right;
    int rows, cols;
    int row_bytes, segment_stages, part_stages, parts;
    const float* more;     // what is added, fp32, as far apart as out's rows; or null
    float* sums;           // fp32 results that go on; or
    char* out;             // the last one, of type `dtype`, times the scale
    Scale scale;
    const float* lost;     // dx: what the rows' targets lost, times their rows of the weight, is added before that; or null
    const int* labels;     // dx: of its rows; or null
    const char* weight;
    int64_t weight_stride, vocabulary;
    int64_t stride;
    int dtype;
};
__device__ __forceinline__ void store_result(float (&v)[8], const GradProductArgs& a, float scale, int i, int j, int valid) {
    if (a.lost) {
        const int label = a.labels[i];
        if (label >= 0 && label < a.vocabulary) {    // what is kept between the passes has been out of these kernels' hands
            const float lost = a.lost[i];
            const char* row = a.weight + (label * a.weight_stride + j) * 2;
            float w[8];
            if (a.dtype == DT_BF16) load_values<DT_BF16>(w, row, valid); else load_values<DT_F16>(w, row, valid);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = fmaf(lost, w[k], v[k]);
        }
    }
    // rows of ignored targets are zeros up to here, and stay so
    const bool none = a.labels && !(fabsf(scale) < __builtin_inff()) && a.labels[i] == kIgnored;
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = none ? v[k] : v[k] * scale;
    const int64_t at = i * a.stride + j;
    if (a.dtype == DT_BF16) store_values<DT_BF16>(v, a.out + at * 2, valid);
    else if (a.dtype == DT_F16) store_values<DT_F16>(v, a.out + at * 2, valid);
    else store_values<DT_F32>(v, a.out + at * 4, valid);
}
struct GradProductOut {
    static constexpr bool kColumns = false;
    const GradProductArgs& a;
    int64_t part;
    float scale;    // read once: behind a store every piece would wait for it again
    struct In { f32x4 lo, hi; };
    __device__ __forceinline__ void begin(int) const {}
    __device__ __forceinline__ void load(int i, int j, In& in) const {
        in.lo = in.hi = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (!a.more || i >= a.rows || j >= a.cols) return;
        float v[8];
        load_values<DT_F32>(v, a.more + i * a.stride + j, a.cols - j);
        in.lo = f32x4{v[0], v[1], v[2], v[3]};
        in.hi = f32x4{v[4], v[5], v[6], v[7]};
    }
    __device__ __forceinline__ void row(int i, int j, const In& in, float (&v)[8]) const {
        if (i >= a.rows || j >= a.cols) return;
#pragma unroll
        for (int k = 0; k < 4; ++k) { v[k] += in.lo[k]; v[4 + k] += in.hi[k]; }
        if (a.out) store_result(v, a, scale, i, j, a.cols - j);
        else store_values<DT_F32>(v, a.sums + part * a.rows * a.stride + i * a.stride + j, a.cols - j);
    }
};
// TURNED: the left operand comes by columns too (dW = G' x).  Bound by the matrix cores: dx of 8192 x 4096 over 16128 in 777 us (1390 TFLOP/s), dW the same sizes in 805.  With operands
// turned by launches of their own instead of by their reads (64 us a piece, and G written twice) the loss of 1003 x 1000 over 32003 took 496 us, so 398.
template <class Product, bool TURNED, int WT, int STAGES> __global__ __launch_bounds__(256, WT >= 96 ? 1 : 2) void grad_product_kernel(GradProductArgs a) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef GemmTile<Product, WT, STAGES, TURNED, true> Tile;
    const int down = (a.rows + Tile::kTile - 1) / Tile::kTile, across = (a.cols + Tile::kTile - 1) / Tile::kTile;
    const int64_t t = tile_of_seat(blockIdx.x & 7, blockIdx.x >> 3, (int64_t)down * across * a.parts);
    if (t < 0) return;
    const int part = (int)(t / (down * across));
    int i, j;
    tile_at((int)(t - (int64_t)part * down * across), down, across, i, j);
    GradProductOut out{a, part, a.out ? a.scale.value() : 1.0f};
    Tile tile(smem);
    tile.segment_stages = a.segment_stages;
    tile.first_stage = part * a.part_stages;
    tile.multiply(a.left, a.right, i * Tile::kTile, j * Tile::kTile, part + 1 < a.parts ? a.part_stages * kStageBytes : a.row_bytes - tile.first_stage * kStageBytes);
    tile.finish(i * Tile::kTile, j * Tile::kTile, out);
}
// The parts' results and `more`, added up in their order.  A thread takes eight values of a row.
__global__ __launch_bounds__(256) void grad_join_kernel(GradProductArgs a, const float* partial) {
    const int pieces = (a.cols + 7) / 8;
    const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x, i = k / pieces;
    const int j = (int)(k - i * pieces) * 8, valid = a.cols - j;
    if (i >= a.rows) return;
    const int64_t at = i * a.stride + j;
    float sum[8];
    load_values<DT_F32>(sum, partial + at, valid);
#pragma unroll 8
    for (int p = 1; p < a.parts; ++p) {
        float v[8];
        load_values<DT_F32>(v, partial + (int64_t)p * a.rows * a.stride + at, valid);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += v[e];
    }
    if (a.more) {
        float v[8];
        load_values<DT_F32>(v, a.more + at, valid);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += v[e];
    }
    if (a.out) store_result(sum, a, a.scale.value(), (int)i, j, valid);
    else store_values<DT_F32>(sum, a.sums + at, valid);
}

}  // namespace fo

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
namespace {
using namespace fo_host;
using fo::u32;

constexpr int64_t kMostWorkgroups = (1 << 24) - 1;    // of 256 threads: a launch has less than 2^32 threads
constexpr int64_t kMostTokens = 1 << 20, kMostCols = 1 << 16, kMostVocabulary = 1 << 24;    // 32-bit offsets into a tile's rows
constexpr int64_t kBlockTokens = 16384;          // rows of one forward launch: bounds the parts' memory
constexpr int64_t kPieceValues = 1 << 27;        // of G in 16 bits: 256 MiB, and up to 256 words of every token more, since pieces are whole multiples of that

// Times of tiles, middle between the three products that write their results (bf16 over 32, 1024 and 2048 values: a 256 x 256 tile takes 19, 46 and 68 us, 192 x 192 -, 32 and
// 46, two 128 x 128 on a compute unit 7, 22 and 36, five 64 x 64 4, 18 and 34, two of those in four stages 3, 9 and 15), and of the logits, whose large tiles have less to do at
// their end (256 x 256 37 and 62 us over 1000 and 2048, 192 x 192 25 and 38).  fp32, where large tiles gain nothing, over 512 and 1024: two 128 x 128 74 and 133 (43 and 74), five 64 x 64 54 and 95 (15 and 24; 15 and 24, 23 and 38).
constexpr fo::TileCost kTileCosts[] = {
    {128, 2, 1, 23.0, 0.0216, 23.0, 0.0216}, {96, 3, 1, 16.5, 0.0150, 16.5, 0.0150}, {64, 2, 2, 6.8, 0.0101, 8.3, 0.0133},
    {32, 2, 5, 3.2, 0.0071, 3.9, 0.0150}, {32, 4, 2, 3.4, 0.0038, 3.4, 0.0060}};
constexpr fo::TileCost kTileCostsLogits[] = {
    {128, 2, 1, 16.0, 0.0216, 16.0, 0.0216}, {96, 3, 1, 10.0, 0.0145, 10.0, 0.0145}, {64, 2, 2, 6.5, 0.0101, 7.5, 0.0133},
    {32, 2, 5, 3.2, 0.0071, 3.9, 0.0150}, {32, 4, 2, 3.4, 0.0038, 3.4, 0.0060}};
constexpr fo::TileCost kTileCostsF32[] = {
    {64, 2, 2, 11.0, 0.061, 14.0, 0.116}, {32, 2, 5, 5.8, 0.0171, 16.0, 0.0765}, {32, 4, 2, 6.5, 0.0168, 7.0, 0.0305}};
struct Costs { const fo::TileCost *first, *last; const fo::TileCost* begin() const { return first; } const fo::TileCost* end() const { return last; } };

int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t aligned(int64_t bytes) { return round_up(bytes, 256); }
// How operands are held: in their own type, or fp32 in three bf16 parts, contracted segment after segment, each of whole stages.
struct Mode {
    int dtype;
    bool in_parts;
    int bytes() const { return dtype == FO_F32 && !in_parts ? 4 : 2; }
    int parts() const { return in_parts ? 3 : 1; }
    int segments() const { return in_parts ? fo::kSegments : 1; }
    int64_t length(int64_t n) const { return round_up(n, in_parts ? 64 : 64 / bytes()); }                     // of an operand's row
    int64_t form(int64_t rows, int64_t inner) const { return aligned(rows * length(inner) * parts() * bytes()); }
    int stages(int64_t values) const { return (int)(values * bytes() / fo::kStageBytes); }
    Costs costs(bool logits = false) const {
        if (dtype == FO_F32 && !in_parts) return {kTileCostsF32, kTileCostsF32 + 3};
        return logits ? Costs{kTileCostsLogits, kTileCostsLogits + 5} : Costs{kTileCosts, kTileCosts + 5};
    }
};

int validate(const char* what, int dtype, int64_t tokens, int64_t cols, int64_t vocabulary) {
    if (tokens < 0 || cols < 0 || vocabulary < 0) return fail(FO_ERR_INVALID_ARGUMENT, "%s: negative size", what);
    if (dtype < FO_F32 || dtype > FO_F16) return fail(FO_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    if (tokens > kMostTokens || cols > kMostCols || vocabulary > kMostVocabulary)
        return fail(FO_ERR_UNSUPPORTED, "%s: %lld tokens of %lld values over a vocabulary of %lld are too many", what, (long long)tokens, (long long)cols, (long long)vocabulary);
    if (tokens == 0 || cols == 0 || vocabulary == 0) return fail(FO_ERR_UNSUPPORTED, "%s: an empty product", what);
    return 0;
}

template <class K, class A> int launch(K kernel, int64_t grid, int threads, int lds, hipStream_t stream, const char* what, const A& args) {
    if (grid > kMostWorkgroups) return fail(FO_ERR_UNSUPPORTED, "%s: %lld workgroups are more than one launch takes", what, (long long)grid);
    if (lds > 65536) {
        if (int rc = check_hip(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds), what)) return rc;
    }
    kernel<<<dim3((unsigned)grid), dim3(threads), lds, stream>>>(args);
    return check_hip(hipGetLastError(), what);
}

// ---- products in tiles of a size that suits the result
fo::TileCost tile_for(const Mode& mode, bool logits, int64_t rows, int64_t cols, double inner, int cus, double* time_of = nullptr) {
    fo::TileCost best{};
    double least = 0.0;
    for (const fo::TileCost& t : mode.costs(logits)) {
        const double time = fo::tiles_time(t, (double)fo::tiles_of(rows, cols, t.wt), inner, cus);
        if (!best.wt || time < least) { best = t; least = time; }
    }
    if (time_of) *time_of = least;
    return best;
}

// fp32 in parts where that takes less: the logits in six times the length with what laying out both operands moves (10 bytes a value, at 4 TB/s) against fp32
// instructions.  With gradients 512 x 1000 over 5003 takes 240 us whole and 302 in parts, 64 x 1024 over 32768 223 and 438, 1024 x 1024 over 8192 599 and 521, 8192 x 4096 over 16000
// 31.3 and 22.8 ms.
Mode mode_of(int dtype, int64_t tokens, int64_t cols, int64_t vocabulary, int cus) {
    if (dtype != FO_F32) return {dtype, false};
    const Mode whole{dtype, false}, parts{dtype, true};
    double by_whole, by_parts;
    (void)tile_for(whole, true, tokens, vocabulary, (double)whole.length(cols), cus, &by_whole);
    (void)tile_for(parts, true, tokens, vocabulary, (double)(parts.length(cols) * parts.segments()), cus, &by_parts);
    by_parts += (double)(tokens + vocabulary) * (double)cols * 10e-6 / 4.0;
    return by_parts < by_whole ? parts : whole;
}

// A product of few tiles over a long contraction is cut along it: parts of whole stages, their fp32 results joined by another launch.  1003 x 1000 over
// 32003 values: 157 us in 64 x 64 tiles, 86 + 6 in parts (the loss with gradients 433 and 366); 64 x 4096 over 128256 1885 and 1367.
struct Cut { fo::TileCost tile; int parts; int64_t part; double time; };
constexpr int kMostParts = 32;
constexpr int64_t kLeastPartValues = 512;
Cut cut_for(const Mode& mode, int64_t rows, int64_t cols, int64_t inner, int cus) {
    Cut best{};
    for (const fo::TileCost& t : mode.costs()) {
        const double tiles = (double)fo::tiles_of(rows, cols, t.wt);
        for (int parts = 1; parts <= kMostParts; parts = parts < 4 ? parts + 1 : parts + parts / 2) {
            if (parts > 1 && inner < parts * kLeastPartValues) break;
            const int64_t part = round_up((inner + parts - 1) / parts, 64), used = (inner + part - 1) / part;
            // the join reads and writes 4 bytes a value and part, at 4 TB/s, and is a launch
            const double join = used > 1 ? 5.0 + (double)used * (double)(rows * cols) * 8e-6 / 4.0 : 0.0;
            const double time = fo::tiles_time(t, tiles * (double)used, (double)part, cus) + join;
            if (!best.parts || time < best.time) best = Cut{t, (int)used, part, time};
        }
    }
    return best;
}

template <class Product> struct LogitsLaunch {
    typedef fo::LogitsArgs Args;
    static constexpr bool kF32 = Product::kBytes == 4;
    template <int WT, int STAGES> static auto kernel() { return fo::logits_kernel<Product, WT, STAGES>; }
    template <int WT, int STAGES> static constexpr int lds() { return fo::GemmTile<Product, WT, STAGES>::kLds; }
    static int64_t rows(const Args& a) { return a.x.rows; }
    static int64_t cols(const Args& a) { return a.weight.rows; }
    static int64_t parts(const Args&) { return 1; }
};
template <int DT, class Product> struct GradLaunch {
    typedef fo::GradArgs Args;
    static constexpr bool kF32 = Product::kBytes == 4;
    template <int WT, int STAGES> static auto kernel() { return fo::grad_kernel<DT, Product, WT, STAGES>; }
    template <int WT, int STAGES> static constexpr int lds() { return fo::GemmTile<Product, WT, STAGES>::kLds; }
    static int64_t rows(const Args& a) { return a.x.rows; }
    static int64_t cols(const Args& a) { return a.weight.rows; }
    static int64_t parts(const Args&) { return 1; }
};
template <class Product, bool TURNED> struct ProductLaunch {
    typedef fo::GradProductArgs Args;
    static constexpr bool kF32 = Product::kBytes == 4;
    template <int WT, int STAGES> static auto kernel() { return fo::grad_product_kernel<Product, TURNED, WT, STAGES>; }
    template <int WT, int STAGES> static constexpr int lds() { return fo::GemmTile<Product, WT, STAGES, TURNED, true>::kLds; }
    static int64_t rows(const Args& a) { return a.rows; }
    static int64_t cols(const Args& a) { return a.cols; }
    static int64_t parts(const Args& a) { return a.parts; }
};

template <class L, int WT, int STAGES> int launch_tiles(const typename L::Args& a, hipStream_t s, const char* what) {
    const int64_t tiles = fo::tiles_of(L::rows(a), L::cols(a), WT) * L::parts(a);
    return launch(L::template kernel<WT, STAGES>(), 8 * fo::seats_of(tiles), 256, L::template lds<WT, STAGES>(), s, what, a);
}
template <class L> int launch_tiles(const fo::TileCost& t, const typename L::Args& a, hipStream_t s, const char* what) {
    if constexpr (!L::kF32) {
        if (t.wt == 128) return launch_tiles<L, 128, 2>(a, s, what);
        if (t.wt == 96) return launch_tiles<L, 96, 3>(a, s, what);
    }
    switch (t.wt) {
        case 64: return launch_tiles<L, 64, 2>(a, s, what);
        default: return t.stages == 4 ? launch_tiles<L, 32, 4>(a, s, what) : launch_tiles<L, 32, 2>(a, s, what);
    }
}

// ---- operands
struct Matrix {
    const char* p;
    int64_t stride, rows, cols;
    int dtype;
    int64_t width() const { return dtype == FO_F32 ? 4 : 2; }
    Matrix part(int64_t first, int64_t n) const { return {p + first * stride * width(), stride, n, cols, dtype}; }
    // Whether the rows can be operand rows where they are: whole pieces, aligned.
    bool ready(const Mode& m) const {
        const int64_t per = 16 / width();
        return !m.in_parts && cols % per == 0 && stride % per == 0 && stride >= 0 && stride < (1 << 22) && ((uintptr_t)p & 15) == 0;
    }
};
// Rows of an operand, `stride` bytes apart.  part_stride, order: see fo_gemm.h.
fo::Operand operand(const void* p, int64_t stride, int64_t rows, int64_t part_stride, u32 order) { return {(const char*)p, stride, nullptr, 0, (int)rows, 0, part_stride, order, 0}; }
// The same whose columns are the operand: `depth` rows of `length` values.
fo::Operand turned(fo::Operand o, int64_t length, int64_t depth) {
    o.rows = (int)length;
    o.depth = (int)depth;
    o.pieces = 0;
    return o;
}

// The rows of m as an operand: in place where they can be and `copy` does not ask for more, else laid out at `space`, filled up to out_rows rows.  labels: see FormArgs.
int operand_of(const Mode& mode, const Matrix& m, bool copy, const int* labels, int64_t out_rows, char* space, u32 order, fo::Operand& to, hipStream_t s, const char* what) {
    const int64_t length = mode.length(m.cols);
    if (m.ready(mode) && !copy) {
        to = operand(m.p, m.stride * m.width(), m.rows, 0, order);
        to.pieces = m.cols == length ? 0 : (int)(m.cols * m.width() / 16);
        return 0;
    }
    const int64_t part_stride = out_rows * length * mode.bytes();
    to = operand(space, length * mode.bytes(), m.rows, part_stride, order);
    const fo::FormArgs a{m.p, space, labels, m.stride, part_stride, (int)m.rows, (int)m.cols, (int)out_rows, (int)length};
    const int64_t grid = (out_rows * (length / 8) + 255) / 256;
    switch (m.dtype) {
        case FO_F32:
            return mode.in_parts ? launch(fo::form_kernel<fo::DT_F32, fo::Bf16PartsProduct>, grid, 256, 0, s, what, a)
                                 : launch(fo::form_kernel<fo::DT_F32, fo::F32Product>, grid, 256, 0, s, what, a);
        case FO_BF16: return launch(fo::form_kernel<fo::DT_BF16, fo::Bf16Product>, grid, 256, 0, s, what, a);
        default: return launch(fo::form_kernel<fo::DT_F16, fo::F16Product>, grid, 256, 0, s, what, a);
    }
}

template <class Product, bool TURNED> int product(const Mode& mode, fo::GradProductArgs a, const Cut& cut, float* partial, hipStream_t s, const char* what) {
    a.parts = cut.parts;
    a.part_stages = mode.stages(cut.part);
    if (cut.parts == 1) return launch_tiles<ProductLaunch<Product, TURNED>>(cut.tile, a, s, what);
    fo::GradProductArgs some = a;
    some.more = nullptr;
    some.out = nullptr;
    some.sums = partial;
    if (int rc = launch_tiles<ProductLaunch<Product, TURNED>>(cut.tile, some, s, what)) return rc;
    const int64_t grid = ((int64_t)a.rows * ((a.cols + 7) / 8) + 255) / 256;
    if (grid > kMostWorkgroups) return fail(FO_ERR_UNSUPPORTED, "%s: too large a result for one launch", what);
    fo::grad_join_kernel<<<dim3((unsigned)grid), dim3(256), 0, s>>>(a, partial);
    return check_hip(hipGetLastError(), what);
}

template <class F> int by_product(const Mode& mode, const F& f) {
    if (mode.in_parts) return f.template run<fo::DT_F32, fo::Bf16PartsProduct>();
    if (mode.dtype == FO_F32) return f.template run<fo::DT_F32, fo::F32Product>();
    return mode.dtype == FO_BF16 ? f.template run<fo::DT_BF16, fo::Bf16Product>() : f.template run<fo::DT_F16, fo::F16Product>();
}

// Compute units to plan for; without a device those of this part, so that sizes can be asked for anywhere.
int units() {
    const int cus = compute_units();
    return cus > 0 ? cus : 256;
}

int check_common(const char* what, const void* x, const void* weight, int reduction, float smoothing, const void* workspace) {
    if (!x || !weight) return fail(FO_ERR_INVALID_ARGUMENT, "%s: x and weight must not be NULL", what);
    if (reduction < FO_REDUCE_NONE || reduction > FO_REDUCE_MEAN) return fail(FO_ERR_INVALID_ARGUMENT, "%s: unknown reduction %d", what, reduction);
    if (!(smoothing >= 0.0f && smoothing <= 1.0f)) return fail(FO_ERR_INVALID_ARGUMENT, "%s: smoothing is between 0 and 1", what);
    if (!workspace || (uintptr_t)workspace & 255) return fail(FO_ERR_INVALID_ARGUMENT, "%s: a workspace, aligned to 256 bytes, is needed", what);
    return 0;
}

// ---- what a call keeps in its workspace
struct ForwardSpace {
    fo::TileCost tile;    // of a full block of tokens
    int64_t rows, parts;
    int64_t picked, losses, stats, sums, x, weight, total;
    ForwardSpace(const Mode& mode, const Matrix& of_x, const Matrix& of_weight, bool smooth, int cus) {
        const int64_t tokens = of_x.rows, length = mode.length(of_x.cols);
        rows = tokens < kBlockTokens ? tokens : kBlockTokens;
        tile = tile_for(mode, true, rows, of_weight.rows, (double)(length * mode.segments()), cus);
        parts = (of_weight.rows + tile.wt - 1) / tile.wt;
        picked = 0;
        losses = picked + aligned(rows * 4);
        stats = losses + aligned(tokens * 4);
        sums = stats + aligned(rows * parts * 8);
        x = sums + (smooth ? aligned(rows * parts * 4) : 0);
        weight = x + (of_x.ready(mode) && of_x.cols == length ? 0 : mode.form(rows, of_x.cols));
        total = weight + (of_weight.ready(mode) ? 0 : mode.form(of_weight.rows, of_weight.cols));
    }
};

struct BackwardSpace {
    int64_t piece;    // tokens of the vocabulary at a time
    int64_t factors, lost, scale, x, weight, grad, sums, partial, total;
    Cut dx_cut, dw_cut;
    // dW reads x with the rows of ignored targets left out; and the logits, where nothing fills up the rows, filled up
    static bool copies(const Mode& mode, const Matrix& of_x, bool dw) { return dw || of_x.cols != mode.length(of_x.cols) || !of_x.ready(mode); }
    BackwardSpace(const Mode& mode, const Matrix& of_x, const Matrix& of_weight, bool dx, bool dw, int cus) {
        const int64_t tokens = of_x.rows, cols = of_x.cols, vocabulary = of_weight.rows;
        const int64_t most = round_up(kPieceValues * 2 / (mode.parts() * mode.bytes()) / tokens + 1, 256);
        const int64_t pieces = (vocabulary + most - 1) / most;
        piece = round_up((vocabulary + pieces - 1) / pieces, 256);
        if (piece > vocabulary) piece = vocabulary;
        // a last piece that is shorter goes by the same cuts: its parts are fewer
        dx_cut = dx ? cut_for(mode, tokens, cols, mode.length(piece) * mode.segments(), cus) : Cut{};
        dw_cut = dw ? cut_for(mode, piece, cols, mode.length(tokens) * mode.segments(), cus) : Cut{};
        factors = 0;
        lost = factors + aligned(tokens * 4);
        scale = lost + aligned(tokens * 4);
        x = scale + 256;
        weight = x + (copies(mode, of_x, dw) ? mode.form(mode.length(tokens), cols) : 0);
        grad = weight + (of_weight.ready(mode) ? 0 : mode.form(piece, cols));
        sums = grad + mode.form(tokens, piece);
        partial = sums + (dx && piece < vocabulary ? aligned(tokens * cols * 4) : 0);
        const int64_t of_dx = dx_cut.parts > 1 ? dx_cut.parts * tokens * cols : 0, of_dw = dw_cut.parts > 1 ? dw_cut.parts * piece * cols : 0;
        total = partial + aligned((of_dx > of_dw ? of_dx : of_dw) * 4);
    }
};

struct Forward {
    Mode mode;
    Matrix x, weight;
    const void* targets;
    int index_bytes, reduction;
    int64_t ignore;
    float smoothing;
    float *loss, *kept;
    char* base;
    const ForwardSpace& at;
    int cus;
    hipStream_t s;

    template <int DT, class Product> int run() const {
        const char* what = "fo_linear_cross_entropy";
        float *most = kept, *log_sum = most + x.rows, *count = log_sum + x.rows;
        int* labels = (int*)(count + 1);
        const fo::Targets t{targets, index_bytes};
        float* losses = reduction == FO_REDUCE_NONE ? loss : (float*)(base + at.losses);
        fo::Operand w;
        if (int rc = operand_of(mode, weight, false, nullptr, weight.rows, base + at.weight, fo::kRightOrder, w, s, what)) return rc;
        const int64_t length = mode.length(x.cols), inner = length * mode.segments();
        const int row_bytes = (int)(inner * mode.bytes()), segment = mode.stages(length);
        for (int64_t first = 0; first < x.rows; first += kBlockTokens) {
            const Matrix some = x.part(first, x.rows - first < kBlockTokens ? x.rows - first : kBlockTokens);
            fo::Operand rows;
            if (int rc = operand_of(mode, some, x.cols != length, nullptr, some.rows, base + at.x, fo::kLeftOrder, rows, s, what)) return rc;
            // a last block is shorter, and its tiles may be smaller only where its parts need no more space
            fo::TileCost tile = tile_for(mode, true, some.rows, weight.rows, (double)inner, cus);
            if (some.rows * ((weight.rows + tile.wt - 1) / tile.wt) > at.rows * at.parts) tile = at.tile;
            const fo::LogitsArgs a{rows, w, row_bytes, segment, t, first, (fo::f32x2*)(base + at.stats), smoothing > 0.0f ? (float*)(base + at.sums) : nullptr, (float*)(base + at.picked)};
            if (int rc = launch_tiles<LogitsLaunch<Product>>(tile, a, s, what)) return rc;
            const fo::JoinArgs join{a.stats, a.sums, a.picked, t, first, ignore, weight.rows, most + first, log_sum + first, losses + first, labels + first, (int)some.rows,
                                    (int)((weight.rows + tile.wt - 1) / tile.wt), smoothing};
            int rc;
            if (some.rows >= 64 * 128) rc = launch(fo::loss_join_kernel<64>, (some.rows + 63) / 64, 1024, 0, s, what, join);
            else if (some.rows >= 64) rc = launch(fo::loss_join_kernel<8>, (some.rows + 7) / 8, 1024, 0, s, what, join);
            else rc = launch(fo::loss_join_kernel<1>, some.rows, 1024, 0, s, what, join);
            if (rc) return rc;
        }
        if (reduction == FO_REDUCE_NONE) return 0;
        fo::loss_reduce_kernel<<<dim3(1), dim3(1024), 0, s>>>(losses, labels, x.rows, reduction, loss, count);
        return check_hip(hipGetLastError(), what);
    }
};

struct Backward {
    Mode mode;
    Matrix x, weight;
    int reduction;
    float smoothing;
    const float *kept, *upstream;
    int64_t upstream_stride;
    char *dx, *dw, *base;
    const BackwardSpace& at;
    int cus;
    hipStream_t s;

    template <int DT, class Product> int run() const {
        const char* what = "fo_linear_cross_entropy_backward";
        const float *most = kept, *log_sum = most + x.rows, *count = log_sum + x.rows;
        const int* labels = (const int*)(count + 1);
        float *sums = (float*)(base + at.sums), *partial = (float*)(base + at.partial), *factors = nullptr;
        float* lost = x.dtype != FO_F32 && dx ? (float*)(base + at.lost) : nullptr;
        const float top = x.dtype == FO_F16 ? 32768.0f : 1.0f;
        fo::Scale scale{upstream, reduction != FO_REDUCE_NONE ? count : nullptr, 1.0f / top, reduction == FO_REDUCE_MEAN};
        // rows of their own losses have factors also where all come back with the same: zeros for ignored rows, so that no product's result needs to know of an infinite one
        if (reduction == FO_REDUCE_NONE || (upstream_stride != 0 && x.rows > 1)) {
            factors = (float*)(base + at.factors);
            float* largest = (float*)(base + at.scale);
            fo::loss_factors_kernel<<<dim3(1), dim3(1024), 0, s>>>(upstream, upstream_stride, labels, x.rows, reduction, count, top, factors, largest);
            if (int rc = check_hip(hipGetLastError(), what)) return rc;
            scale = {largest, nullptr, 1.0f / top, false};
        }
        const int64_t tokens_length = mode.length(x.rows), cols_length = mode.length(x.cols), cols_inner = cols_length * mode.segments();
        fo::Operand rows;
        if (int rc = operand_of(mode, x, BackwardSpace::copies(mode, x, dw != nullptr), labels, tokens_length, base + at.x, fo::kLeftOrder, rows, s, what)) return rc;
        fo::Operand x_turned = turned(rows, cols_length, tokens_length);
        x_turned.order = fo::kRightOrder;
        for (int64_t first = 0; first < weight.rows; first += at.piece) {
            const int64_t n = weight.rows - first < at.piece ? weight.rows - first : at.piece, length = mode.length(n);
            const bool last = first + n == weight.rows;
            const Matrix some = weight.part(first, n);
            fo::Operand w;
            if (int rc = operand_of(mode, some, false, nullptr, n, base + at.weight, fo::kRightOrder, w, s, what)) return rc;
            const fo::Operand g = operand(base + at.grad, length * mode.bytes(), x.rows, x.rows * length * mode.bytes(), fo::kLeftOrder);
            const fo::GradArgs grad{rows, w, (int)(cols_inner * mode.bytes()), mode.stages(cols_length), labels, most, log_sum, factors, top, base + at.grad, lost, g.part_stride, (int)length,
                                    (int)first, 1.0f - smoothing, smoothing / (float)weight.rows};
            if (int rc = launch_tiles<GradLaunch<DT, Product>>(tile_for(mode, false, x.rows, n, (double)cols_inner, cus), grad, s, what)) return rc;
            fo::GradProductArgs p{};
            p.cols = (int)x.cols;
            p.scale = scale;
            p.stride = x.cols;
            p.dtype = x.dtype;
            if (dx) {
                p.left = g;
                p.right = turned(w, some.ready(mode) ? x.cols : cols_length, n);
                p.rows = (int)x.rows;
                p.row_bytes = (int)(length * mode.segments() * mode.bytes());
                p.segment_stages = mode.stages(length);
                p.more = first ? sums : nullptr;
                p.sums = last ? nullptr : sums;
                p.out = last ? dx : nullptr;
                p.lost = lost;
                p.labels = labels;
                p.weight = weight.p;
                p.weight_stride = weight.stride;
                p.vocabulary = weight.rows;
                Cut cut = at.dx_cut;
                cut.parts = (int)((length * mode.segments() + cut.part - 1) / cut.part);
                if (int rc = product<Product, false>(mode, p, cut, partial, s, what)) return rc;
            }
            if (dw) {
                p.left = turned(g, length, x.rows);
                p.right = x_turned;
                p.rows = (int)n;
                p.row_bytes = (int)(tokens_length * mode.segments() * mode.bytes());
                p.segment_stages = mode.stages(tokens_length);
                p.labels = nullptr;
                p.more = nullptr;
                p.sums = nullptr;
                p.out = dw + first * x.cols * x.width();
                p.lost = nullptr;
                if (int rc = product<Product, true>(mode, p, at.dw_cut, partial, s, what)) return rc;
            }
        }
        return 0;
    }
};

}  // namespace

extern "C" {

int64_t fo_linear_cross_entropy_workspace(const void* x, int dtype, int64_t tokens, int64_t x_stride, const void* weight, int64_t weight_stride, int64_t vocabulary, int64_t cols,
                                          float smoothing) {
    if (int rc = validate("fo_linear_cross_entropy", dtype, tokens, cols, vocabulary)) return rc;
    const int cus = units();
    return ForwardSpace(mode_of(dtype, tokens, cols, vocabulary, cus), {(const char*)x, x_stride, tokens, cols, dtype}, {(const char*)weight, weight_stride, vocabulary, cols, dtype},
                        smoothing > 0.0f, cus).total;
}

int fo_linear_cross_entropy(const void* x, int dtype, int64_t tokens, int64_t x_stride, const void* weight, int64_t weight_stride, int64_t vocabulary, int64_t cols,
                            const void* targets, int index_bytes, int64_t ignore, int reduction, float smoothing, float* loss, float* kept, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    const char* what = "fo_linear_cross_entropy";
    if (int rc = validate(what, dtype, tokens, cols, vocabulary)) return rc;
    if (int rc = check_common(what, x, weight, reduction, smoothing, workspace)) return rc;
    if (!targets || !loss || !kept) return fail(FO_ERR_INVALID_ARGUMENT, "%s: targets, loss and kept must not be NULL", what);
    if (index_bytes != 4 && index_bytes != 8) return fail(FO_ERR_INVALID_ARGUMENT, "%s: targets of %d bytes", what, index_bytes);
    const int cus = units();
    const Mode mode = mode_of(dtype, tokens, cols, vocabulary, cus);
    const Matrix of_x{(const char*)x, x_stride, tokens, cols, dtype}, of_weight{(const char*)weight, weight_stride, vocabulary, cols, dtype};
    const ForwardSpace at(mode, of_x, of_weight, smoothing > 0.0f, cus);
    if (workspace_bytes < at.total) return fail(FO_ERR_INVALID_ARGUMENT, "%s: workspace too small", what);
    const Forward f{mode, of_x, of_weight, targets, index_bytes, reduction, ignore, smoothing, loss, kept, (char*)workspace, at, cus, (hipStream_t)stream};
    return by_product(mode, f);
}

int64_t fo_linear_cross_entropy_backward_workspace(const void* x, int dtype, int64_t tokens, int64_t x_stride, const void* weight, int64_t weight_stride, int64_t vocabulary,
                                                   int64_t cols, int want_dx, int want_dw) {
    if (int rc = validate("fo_linear_cross_entropy_backward", dtype, tokens, cols, vocabulary)) return rc;
    const int cus = units();
    return BackwardSpace(mode_of(dtype, tokens, cols, vocabulary, cus), {(const char*)x, x_stride, tokens, cols, dtype}, {(const char*)weight, weight_stride, vocabulary, cols, dtype},
                         want_dx != 0, want_dw != 0, cus).total;
}

int fo_linear_cross_entropy_backward(const void* x, int dtype, int64_t tokens, int64_t x_stride, const void* weight, int64_t weight_stride, int64_t vocabulary,
                                     int64_t cols, int reduction, float smoothing, const float* kept, const float* upstream, int64_t upstream_stride, void* dx, void* dw,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "fo_linear_cross_entropy_backward";
    if (int rc = validate(what, dtype, tokens, cols, vocabulary)) return rc;
    if (int rc = check_common(what, x, weight, reduction, smoothing, workspace)) return rc;
    if (!kept || !upstream || (!dx && !dw)) return fail(FO_ERR_INVALID_ARGUMENT, "%s: kept, upstream and a result must be given", what);
    const int cus = units();
    const Mode mode = mode_of(dtype, tokens, cols, vocabulary, cus);
    const Matrix of_x{(const char*)x, x_stride, tokens, cols, dtype}, of_weight{(const char*)weight, weight_stride, vocabulary, cols, dtype};
    const BackwardSpace at(mode, of_x, of_weight, dx != nullptr, dw != nullptr, cus);
    if (workspace_bytes < at.total) return fail(FO_ERR_INVALID_ARGUMENT, "%s: workspace too small", what);
    const Backward b{mode, of_x, of_weight, reduction, smoothing, kept, upstream, upstream_stride, (char*)dx, (char*)dw, (char*)workspace, at, cus, (hipStream_t)stream};
    return by_product(mode, b);
}

}  // extern "C"
