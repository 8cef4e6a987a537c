// Newton-Schulz orthogonalisation of matrices and the Muon optimizer step around it, for gfx950, with their C entry points.
//
// Mathematics.  For a matrix G (rows x cols; its shorter side m, its longer n; X is G with the shorter side as rows):
//     X <- G / (|G|_F + eps),  then `steps` times  S = X X',  B = b S + c S S,  X <- a X + B X.
// The polynomial drives every singular value towards one and leaves the singular vectors alone.
//
// Precision.  The products run on the matrix cores in fp16 with fp32 sums.  Rounding X itself to fp16 in every step would
// cost up to 1e-2 of the result: an error among the small singular directions is multiplied like the signal there (3.4 per
// step).  So X is held in two parts, hi (fp16, the operand of the products) and lo (bf16, the rest, 19 bits or more together); lo
// enters where X is multiplied by a.  The diagonals of S and B, by far their largest entries on a flat spectrum, are kept apart
// in fp32; the products see the matrices without them: S S = O O + O D + D O + D D for S = O + D, and B's is added to a.  What is left (S and B off the diagonal and the products' X
// in fp16) costs 1e-4 .. 1.3e-3 of the result, below the bfloat16 rounding it is handed out with; the smallest matrices are done in fp32.  X starts at |X|_F = 1, entries as small as 1e-4, so
// the first X is kept times a power of two near sqrt(n), in fp16's normal range.
//
// Layout.  "Main" arrays have G's own orientation, padded with zeros to multiples of 64 (Rp x Cp), a shorter side of at most 32 to 32 (49
// of 23 x 4934 took 195 us with it and 222 with 64), so that the products need no bounds inside; T is hi transposed.  Every product is then rows times rows (fo_gemm.h):
//     S = rows of X by rows of X          (X = hi where rows <= cols, else T); the tiles on and above the diagonal, written twice
//     B = rows of S by rows of S          (S is symmetric); likewise
//     X = rows of B by rows of T          (rows <= cols), or rows of hi by rows of B: main orientation either way
// so the result comes out in G's orientation and the last product's epilogue writes it, or updates the weights with it.
//
// The first two steps of a matrix that is longer than wide are merged: with P = a + B its second S is P S P, so both B's come of
// side x side products and X is read and written once for  X <- P2 P1 X.  That costs three such products more and saves an S
// and a step, 2 longer / shorter times as much arithmetic each; and it costs no accuracy, unlike merging later steps (there an
// error of S is no longer small against the small singular values: 2 to 3 times the error, measured on flat, low-rank, peaked
// and decaying spectra).
//
// One launch covers matrices of many shapes: the shapes travel as kernel arguments, matrices of one shape lie one after the
// other in the workspace.
#include "fo_gemm.h"
#include "fo_host.h"
#include "fo_step.h"

#include <algorithm>
#include <cmath>

namespace fo {

constexpr int kMaxShapes = 16;    // of one launch
constexpr int kPad = 64, kNarrow = 32;
constexpr int kChunk = 8192;      // elements of a matrix whose squares one workgroup sums

// What a matrix is multiplied by for its norm, the power of two first: fp32 holds both for every norm that fp32 values have.
struct Scaling { float power, factor; };

// The matrices of one shape.
struct MatrixGroup {
    int rows, cols, padded_rows, padded_cols, count;
    int first;            // matrix number of the first of them
    int generation;       // of hi and T that X is in
    int chunks;           // sums of squares of each
    int parts;            // S: runs of the long axis that are summed apart
    float unit;           // the power of two that the first X is kept times
    float lr;             // optimizer step: learning rate with the shape's factor
    char* workspace;      // their arrays, see the functions below

    __host__ __device__ bool tall() const { return rows > cols; }
    __host__ __device__ int side() const { return tall() ? padded_cols : padded_rows; }
    __host__ __device__ int64_t area() const { return (int64_t)padded_rows * padded_cols; }
    __host__ __device__ int64_t gram_area() const { return (int64_t)side() * side(); }
    // per matrix: two generations of hi and of T, lo, three square matrices, their diagonals, what normalises, sums of squares.
    // The update before its normalisation (fp32) lies over the second generation, which is written later.
    __host__ __device__ int64_t bytes_each() const {
        return area() * 10 + gram_area() * 6 + (side() * 12 + 255) / 256 * 256 + 256 + ((int64_t)chunks * 8 + 255) / 256 * 256;
    }
    __device__ char* of(int k) const { return workspace + bytes_each() * k; }
    __device__ _Float16* hi(int k, int generation) const { return (_Float16*)(of(k) + generation * area() * 4); }
    __device__ _Float16* t(int k, int generation) const { return (_Float16*)(of(k) + generation * area() * 4 + area() * 2); }
    __device__ float* update(int k) const { return (float*)(of(k) + area() * 4); }
    // Sums over the parts, side x side each: over the generation that the step writes next.
    __host__ __device__ int most_parts() const { return (tall() ? padded_rows : padded_cols) / side(); }
    __device__ float* partial(int k, int part) const { return (float*)(of(k) + (generation ^ 1) * area() * 4) + gram_area() * part; }
    __device__ u32* lo(int k) const { return (u32*)(of(k) + area() * 8); }   // pairs of bf16
    __device__ _Float16* square(int k, int which) const { return (_Float16*)(of(k) + area() * 10 + gram_area() * 2 * which); }
    __device__ float* diagonal(int k, int which) const { return (float*)(of(k) + area() * 10 + gram_area() * 6) + side() * which; }
    __device__ Scaling* scaling(int k) const { return (Scaling*)diagonal(k, 3); }
    __device__ double* squares(int k) const { return (double*)((char*)scaling(k) + 256); }
};

// A launch over all groups.  Workgroups begin[g] .. begin[g + 1] belong to group g; in the products' launches these are seats,
// of which each of the eight dies has all (fo_gemm.h), so that every die gets its share of every shape.
struct Groups {
    MatrixGroup group[kMaxShapes];
    int64_t begin[kMaxShapes + 1];
    int n;
};

__device__ __forceinline__ int group_of(const Groups& a, int64_t b) {
    int g = 0;
    while (g + 1 < a.n && b >= a.begin[g + 1]) ++g;
    return g;
}

// ------------------------------------------------------------------------------------------------
// what comes before the products: momentum, norm, normalised parts
// ------------------------------------------------------------------------------------------------

// Matrices in memory: `stride` elements between those of a stack, `row_stride` between rows, columns adjacent.  Without
// data: the update that the momentum kernel left in the workspace.
struct MatrixSource {
    const void* data;
    int64_t stride, row_stride;
};

template <int DT> __device__ __forceinline__ void read8(const char* p, int valid, float (&v)[8]) {
    constexpr int B = DTypeInfo<DT>::bytes, EPL = 16 / B;
    Pack<B, EPL> raw[B / 2];
#pragma unroll
    for (int i = 0; i < B / 2; ++i) load_piece<B, EPL>(raw[i], p + i * 16, valid - i * EPL);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = widen<DT, EPL>(raw[k / EPL], k % EPL);
}

__device__ __forceinline__ double workgroup_sum(double x, double* lds) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) x += __shfl_down(x, d);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

// Whether a sum of a few squares in fp32 will do: it is not beyond that, nor so small that some of the squares are (what is lost among them is 2^-46
// of a sum of 2^-80).  fp64 holds the square of every fp32 value.
__device__ __forceinline__ bool holds_squares(float sum) { return sum > 0x1p-80f && sum < __builtin_inff(); }
template <int N> __device__ __forceinline__ double sum_of_squares(const float (&v)[N]) {
    float quick = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) quick = fmaf(v[e], v[e], quick);
    if (holds_squares(quick)) return (double)quick;
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < N; ++e) sum = fma((double)v[e], (double)v[e], sum);
    return sum;
}

// The first of what a matrix of this norm is multiplied by.
__device__ __forceinline__ float power_for(double norm) {
    const float near = (float)norm;
    return near > 0x1p64f ? 0x1p-64f : near < 0x1p-64f ? 0x1p64f : 1.0f;
}

// Sum of the squares of a run of 8-value pieces of the matrix, one number per workgroup (in order, so a step repeats to
// the bit).  One read of the matrix, bound by memory: 14336 x 4096 bf16 in 26 to 31 us, 3.8 to 4.5 TB/s.
template <int DT> __global__ __launch_bounds__(256) void squares_kernel(Groups a, MatrixSource source) {
    __shared__ double lds[4];
    const int g = group_of(a, blockIdx.x);
    const MatrixGroup& m = a.group[g];
    const int64_t local = blockIdx.x - a.begin[g];
    const int k = (int)(local / m.chunks), chunk = (int)(local % m.chunks);
    const int64_t pieces = (m.cols + 7) / 8, all = pieces * m.rows, each = (all + m.chunks - 1) / m.chunks;
    const int64_t last = (chunk + 1) * each < all ? (chunk + 1) * each : all;
    double sum = 0.0;
    for (int64_t i = chunk * each + threadIdx.x; i < last; i += 256) {
        const int64_t row = i / pieces;
        const int col = (int)(i - row * pieces) * 8;
        float v[8];
        read8<DT>((const char*)source.data + (source.stride * k + source.row_stride * row + col) * DTypeInfo<DT>::bytes, m.cols - col, v);
        sum += sum_of_squares(v);
    }
    const double total = workgroup_sum(sum, lds);
    if (threadIdx.x == 0) m.squares(k)[chunk] = total;
}

// unit / (|G|_F + eps) of every matrix, one workgroup each: a launch's latency, 5 us.
__global__ __launch_bounds__(256) void norm_kernel(Groups a, float eps) {
    __shared__ double lds[4];
    const int g = group_of(a, blockIdx.x);
    const MatrixGroup& m = a.group[g];
    const int k = (int)(blockIdx.x - a.begin[g]);
    double sum = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < m.chunks; i += 256) sum += m.squares(k)[i];
    const double total = workgroup_sum(sum, lds);
    if (threadIdx.x == 0) {
        const double norm = sqrt(total) + (double)eps;
        const float power = power_for(norm);
        *m.scaling(k) = {power, (float)((double)m.unit / (norm * (double)power))};
    }
}

// Says that a value is rounded to fp32 here.  Left to itself the compiler joins the product or sum that makes it and its conversion to fp16 into one
// instruction, which rounds once, for some uses of a value and in some kernels only.  In the polynomial's 256 x 256 tiles an entry and
// its mirror image then differed by a unit of fp16 at one place in 1e5, and both from what other tiles make.
__device__ __forceinline__ void rounded(float& x) { asm("" : "+v"(x)); }
__device__ __forceinline__ f16x8 half8(const float (&v)[8]) {
    f16x8 h;
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = (_Float16)v[e];
    return h;
}

// 64 x 64 pieces of G, normalised, as hi and lo in G's orientation and hi transposed (through LDS), zeros in the padding.  Bound by
// memory, 6 bytes written per element: 14336 x 4096 bf16 in 84 to 92 us, 5.1 to 5.6 TB/s.
template <int DT> __global__ __launch_bounds__(256) void split_kernel(Groups a, MatrixSource source) {
    __shared__ _Float16 lds[64][64 + 2];
    const int g = group_of(a, blockIdx.x);
    const MatrixGroup& m = a.group[g];
    const int tile_cols = (m.padded_cols + 63) / 64, tiles = (m.padded_rows + 63) / 64 * tile_cols;
    const int64_t local = blockIdx.x - a.begin[g];
    const int k = (int)(local / tiles), tile = (int)(local % tiles);
    const int row0 = tile / tile_cols * 64, col0 = tile % tile_cols * 64;
    const Scaling scale = *m.scaling(k);
    const char* base = source.data ? (const char*)source.data + source.stride * k * DTypeInfo<DT>::bytes : (const char*)m.update(k);
    const int64_t row_stride = source.data ? source.row_stride : m.cols;
    const int piece = (threadIdx.x & 7) * 8;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int r = (threadIdx.x >> 3) + 32 * p, row = row0 + r, col = col0 + piece;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (row < m.rows && col < m.cols) read8<DT>(base + (row_stride * row + col) * DTypeInfo<DT>::bytes, m.cols - col, v);
        f16x8 hi;
        u32x4 lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = v[e] * scale.power * scale.factor;
            rounded(v[e]);
            hi[e] = (_Float16)v[e];
            v[e] -= (float)hi[e];
            lds[r][piece + e] = hi[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f32x2 pair = {v[2 * e], v[2 * e + 1]};
            lo[e] = __builtin_bit_cast(u32, __builtin_convertvector(pair, bf16x2));
        }
        if (row >= m.padded_rows || col >= m.padded_cols) continue;
        const int64_t at = (int64_t)row * m.padded_cols + col;
        *reinterpret_cast<f16x8*>(m.hi(k, 0) + at) = hi;
        *reinterpret_cast<u32x4*>(m.lo(k) + at / 2) = lo;
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int c = (threadIdx.x >> 3) + 32 * p;
        if (col0 + c >= m.padded_cols || row0 + piece >= m.padded_rows) continue;
        f16x8 t;
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = lds[piece + e][c];
        *reinterpret_cast<f16x8*>(m.t(k, 0) + (int64_t)(col0 + c) * m.padded_rows + row0 + piece) = t;
    }
}

// Momentum of the optimizer step, over the flat elements of every matrix (groups of 32 codes run on across rows):
//     m <- mu m + (1 - mu) g,   u = nesterov ? (1 - mu) g + mu m : m
// each product and sum rounded, requantised as the SGD / Lion kernels do (how codes are read: see the kernel); u goes to the workspace in fp32 together with the
// sum of its squares.  Bound by memory: 8 bytes per bf16 element, 218e6 of them in 311 us, 5.6 TB/s.
struct MomentumArgs {
    const fo_tensor_desc* matrices;
    float mu, one_minus_mu;
    int nesterov;
};

template <int DT, bool QUANT, int MODE>
__device__ __forceinline__ double momentum_span(const fo_tensor_desc& d, float* update, Where w, int64_t n, const MomentumArgs& h, const float* lut) {
    constexpr int EPL = DTypeInfo<DT>::epl, PB = DTypeInfo<DT>::bytes, SB = QUANT ? 1 : PB;
    Pack<PB, EPL> g;
    Pack<SB, EPL> raw;
    load_lane<PB, EPL, MODE>(g, d.grad, w, n);
    load_lane<SB, EPL, MODE>(raw, d.mom, w, n);
    const bool live = MODE == kVector || w.first() < n;
    float scale = 1.0f;
    if constexpr (QUANT) { if (live) scale = f16_bits_to_f32(load_scale((const uint16_t*)d.mom_scales, w)); }
    float m[EPL], u[EPL], am = 0.0f;
#pragma unroll
    for (int k = 0; k < EPL; ++k) {
        const float gk = widen<DT, EPL>(g, k) * h.one_minus_mu;
        float old;
        if constexpr (QUANT) old = lookup_mom(lut, byte_of<EPL>(raw, k)) * scale; else old = widen<DT, EPL>(raw, k);
        m[k] = old * h.mu + gk;
        u[k] = h.nesterov ? gk + m[k] * h.mu : m[k];
        am = fmaxf(am, fabsf(m[k]));
    }
    if constexpr (QUANT) {
        am = fmaxf(group_max<EPL>(am), 1e-12f);
        if constexpr (EPL == 8) quantize_mom_quick_verified<EPL>(m, am, raw);
        else quantize_mom(m, am, raw);
        if (live && (threadIdx.x & (32 / EPL - 1)) == 0) store_scale((uint16_t*)d.mom_scales, w, f32_to_f16_bits(am));
    } else {
        narrow_all<DT, EPL>(m, raw);
    }
    store_lane<SB, EPL, MODE>(raw, d.mom, w, n);
    // the update is read again at once: ordinary stores
    float* out = update + w.first();
    if (MODE == kVector || w.first() + EPL <= n) {
#pragma unroll
        for (int k = 0; k < EPL; k += 4) *reinterpret_cast<f32x4*>(out + k) = f32x4{u[k], u[k + 1], u[k + 2], u[k + 3]};
    } else {
#pragma unroll
        for (int k = 0; k < EPL; ++k) {
            if (w.first() + k < n) out[k] = u[k]; else u[k] = 0.0f;
        }
    }
    return sum_of_squares(u);
}

template <int DT, bool QUANT> __global__ __launch_bounds__(256) void momentum_kernel(Groups a, MomentumArgs h) {
    constexpr int EPL = DTypeInfo<DT>::epl;
    __shared__ double lds[4];
    __shared__ __attribute__((aligned(16))) float lut[256];
    const int g = group_of(a, blockIdx.x);
    const MatrixGroup& m = a.group[g];
    const int64_t local = blockIdx.x - a.begin[g], n = (int64_t)m.rows * m.cols;
    const int k = (int)(local / m.chunks), chunk = (int)(local % m.chunks);
    const fo_tensor_desc d = h.matrices[m.first + k];
    if constexpr (QUANT) {
        // (q / 127) / (2 - |q / 127|), the first quotient as torch divides by a number on the GPU, by its reciprocal: 16 of 255 codes are read a
        // unit in the last place beside the step kernels' table and the dequantiser.  With their quotient 56 of 218e6 codes come out one
        // step apart from the same step in elementary torch operations, with this one none.
        const float y = (float)(int8_t)threadIdx.x * (1.0f / 127.0f);
        lut[threadIdx.x] = y / (2.0f - fabsf(y));
        __syncthreads();
    }
    const bool aligned = (((uintptr_t)d.grad | (uintptr_t)d.mom) & 15) == 0;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    double sum = 0.0;
    for (int i = wave; i < kChunk / (64 * EPL); i += 4) {
        const Where w{(int64_t)chunk * kChunk + i * 64 * EPL, (int)(threadIdx.x & 63) * EPL};
        if (w.span >= n) break;
        if (aligned && w.span + 64 * EPL <= n) sum += momentum_span<DT, QUANT, kVector>(d, m.update(k), w, n, h, lut);
        else if (aligned) sum += momentum_span<DT, QUANT, kLane>(d, m.update(k), w, n, h, lut);
        else sum += momentum_span<DT, QUANT, kGuarded>(d, m.update(k), w, n, h, lut);
    }
    const double total = workgroup_sum(sum, lds);
    if (threadIdx.x == 0) m.squares(k)[chunk] = total;
}

// ------------------------------------------------------------------------------------------------
// the products
// ------------------------------------------------------------------------------------------------

// One of a matrix's three square matrices: S, of which `first` says that X still carries the unit (kGram); from two others, out = gamma U V +
// alpha U + beta V (kMixed); or, where U = V and beta = 0, the same with half of the epilogue's reads (kPoly).
// kPartial: S over one part of the long axis, added up by gather_kernel.
enum { kGram, kPoly, kMixed, kPartial };
struct SquareArgs {
    int u, v, out;
    float alpha, beta, gamma;
    int first;
};
// X <- a X + (square matrix `poly`) X, between the given rows and columns of the padded matrices (to their ends at most).
struct StepArgs {
    float a;
    int poly, first;
    int row_begin = 0, col_begin = 0, row_end = INT32_MAX, col_end = INT32_MAX;
};


// Square matrices without their diagonals: all are symmetric, so each tile off the diagonal is written twice.  Of what lies on it both halves are computed.
// Those of S and of its polynomial agree to the bit; those of U V do only as far as U and V commute.  So that no result goes by the tile, which
// all that shares the launch has a say in, it is blocks of 64 x 64 on the diagonal of which both halves are kept, and in larger tiles what is
// below these is copied as well.
template <int KIND, int TILE> struct SymmetricOut {
    static constexpr bool kColumns = true;
    static constexpr bool kCopied = KIND == kMixed && TILE > kPad;
    __device__ __forceinline__ static bool below(int i, int j) { return i / kPad > j / kPad; }
    const _Float16 *u, *v;
    const float *u_diagonal, *v_diagonal;
    _Float16* out;
    float* diagonal;
    int side;
    float scale, alpha, beta, gamma;
    bool mirror;
    float d[8];                   // V's diagonal at the lane's columns

    struct In { f16x8 u, v; float d; };
    __device__ __forceinline__ void begin(int j) {
        if constexpr (KIND != kGram) {
            if (j < side) {
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = v_diagonal[j + e];
            }
        }
    }
    __device__ __forceinline__ void load(int i, int j, In& in) const {
        if constexpr (KIND != kGram) {
            if (i < side && j < side) {
                in.u = *reinterpret_cast<const f16x8*>(u + (int64_t)i * side + j);
                if constexpr (KIND == kMixed) in.v = *reinterpret_cast<const f16x8*>(v + (int64_t)i * side + j);
                in.d = u_diagonal[i];
            }
        }
    }
    __device__ __forceinline__ void row(int i, int j, const In& in, float (&x)[8]) const {
        if (i >= side || j >= side || (kCopied && !mirror && below(i, j))) return;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (KIND == kGram) {
                x[e] *= scale;
                if (i == j + e) { diagonal[i] = x[e]; x[e] = 0.0f; }
            } else if constexpr (KIND == kPoly) {
                const float a = (float)in.u[e];   // 0 on the diagonal
                x[e] = fmaf(gamma, fmaf(in.d + d[e], a, x[e]), alpha * a);
                if (i == j + e) {
                    diagonal[i] = fmaf(in.d, fmaf(gamma, in.d, alpha), x[e]);
                    x[e] = 0.0f;
                }
            } else {
                const float a = (float)in.u[e], b = (float)in.v[e], product = fmaf(in.d, b, fmaf(a, d[e], x[e]));   // a = b = 0 on the diagonal
                x[e] = fmaf(gamma, product, fmaf(alpha, a, beta * b));
                if (i == j + e) {
                    diagonal[i] = fmaf(gamma, fmaf(in.d, d[e], product), fmaf(alpha, in.d, beta * d[e]));
                    x[e] = 0.0f;
                }
            }
            rounded(x[e]);
        }
        *reinterpret_cast<f16x8*>(out + (int64_t)i * side + j) = half8(x);
    }
    __device__ __forceinline__ bool columns() const { return kCopied || mirror; }
    __device__ __forceinline__ void column(int i, int j, const float (&x)[8]) const {
        if (i >= side || j >= side || (kCopied && !mirror && !below(j, i))) return;
        *reinterpret_cast<f16x8*>(out + (int64_t)j * side + i) = half8(x);
    }
};

struct PartialOut {
    static constexpr bool kColumns = false;
    float* out;
    int side;
    struct In {};
    __device__ __forceinline__ void begin(int) const {}
    __device__ __forceinline__ void load(int, int, In&) const {}
    __device__ __forceinline__ void row(int i, int j, In, const float (&x)[8]) const {
        if (i >= side || j >= side) return;
        f32x4* to = reinterpret_cast<f32x4*>(out + (int64_t)i * side + j);
        to[0] = f32x4{x[0], x[1], x[2], x[3]};
        to[1] = f32x4{x[4], x[5], x[6], x[7]};
    }
};

// Bound by the matrix cores, with 192 x 192 tiles as much by LDS: S of 14336 x 4096 in 272 us (885 TFLOP/s of the half that is computed), a
// square of 4096 x 4096 in 95 (medians of an iteration's launches, whose products pull the clock down; 232 and 81 at least; one round of 253
// tiles either way; 256 x 256 tiles would fill 136 of 256 compute units).
template <int WT, int STAGES, int KIND> __global__ __launch_bounds__(256, WT >= 96 ? 1 : 2) void symmetric_kernel(Groups a, SquareArgs h) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef GemmTile<F16Product, WT, STAGES> Tile;
    const int64_t seat = blockIdx.x >> 3;
    const int g = group_of(a, seat);
    const MatrixGroup& m = a.group[g];
    const int side = m.side(), n = (side + Tile::kTile - 1) / Tile::kTile, tiles = n * (n + 1) / 2;
    const int parts = KIND == kPartial ? m.parts : 1, each = tiles * parts;
    const int64_t local = tile_of_seat(blockIdx.x & 7, seat - a.begin[g], (int64_t)each * m.count);
    if (local < 0) return;
    const int k = (int)(local / each), part = (int)(local % each) / tiles;
    int i, j;
    tile_at_symmetric((int)(local % tiles), n, i, j);
    const bool tall = m.tall();
    const _Float16* x = tall ? m.t(k, m.generation) : m.hi(k, m.generation);
    constexpr bool kOfX = KIND == kGram || KIND == kPartial;
    const int64_t length = (kOfX ? (tall ? m.padded_rows : m.padded_cols) : side) * 2;
    // whole stages of 64 values for each part
    const int64_t run = KIND == kPartial ? ((length / kStageBytes + parts - 1) / parts) * kStageBytes : length, from = part * run;
    const Operand left{(const char*)(kOfX ? x : m.square(k, h.u)) + from, length, nullptr, 0, side};
    const Operand right{(const char*)(kOfX ? x : m.square(k, h.v)) + from, length, nullptr, 0, side};
    Tile tile(lds);
    tile.multiply(left, right, i * Tile::kTile, j * Tile::kTile, (int)(run < length - from ? run : length - from));
    if constexpr (KIND == kPartial) {
        PartialOut out{m.partial(k, part), side};
        tile.finish(i * Tile::kTile, j * Tile::kTile, out);
    } else {
        SymmetricOut<KIND, Tile::kTile> out{m.square(k, h.u), m.square(k, h.v), m.diagonal(k, h.u), m.diagonal(k, h.v), m.square(k, h.out), m.diagonal(k, h.out), side,
                               h.first ? 1.0f / (m.unit * m.unit) : 1.0f, h.alpha, h.beta, h.gamma, i != j, {}};
        tile.finish(i * Tile::kTile, j * Tile::kTile, out);
    }
}

// S of its parts, in order; a workgroup takes four rows of a 64 x 64 tile on or above the diagonal, a thread an entry, so that the
// loads of many parts are under way at once.
__global__ __launch_bounds__(256) void gather_kernel(Groups a, SquareArgs h) {
    const int g = group_of(a, blockIdx.x);
    const MatrixGroup& m = a.group[g];
    const int side = m.side(), n = (side + 63) / 64, each = n * (n + 1) / 2 * 16;
    const int64_t local = blockIdx.x - a.begin[g];
    const int k = (int)(local / each), piece = (int)(local % each);
    int i, j;
    tile_at_symmetric(piece / 16, n, i, j);
    i = i * 64 + piece % 16 * 4 + (threadIdx.x >> 6);
    j = j * 64 + (threadIdx.x & 63);
    if (i > j || j >= side) return;
    const float* in = m.partial(k, 0) + (int64_t)i * side + j;
    float x = 0.0f;
#pragma unroll 8
    for (int part = 0; part < m.parts; ++part) x += in[m.gram_area() * part];
    if (h.first) x *= 1.0f / (m.unit * m.unit);
    if (i == j) { m.diagonal(k, h.out)[i] = x; x = 0.0f; }
    _Float16* s = m.square(k, h.out);
    rounded(x);
    s[(int64_t)i * side + j] = s[(int64_t)j * side + i] = (_Float16)x;
}

// X <- a X + B X, common to the steps: x = (acc + (a + d) (hi + lo)) / unit, d the diagonal entry of B.
struct ApplyIn {
    const _Float16* hi;
    u32* lo;
    const float* diagonal;
    int rows, cols;     // padded
    float a, scale;
    bool tall;
    float d[8];         // of the lane's columns

    struct In { f16x8 hi; u32x4 lo; float d; };
    __device__ __forceinline__ void begin(int j) {
        if (tall && j < cols) {
#pragma unroll
            for (int e = 0; e < 8; ++e) d[e] = a + diagonal[j + e];
        }
    }
    __device__ __forceinline__ void load(int i, int j, In& in) const {
        if (i >= rows || j >= cols) return;
        const int64_t at = (int64_t)i * cols + j;
        in.hi = *reinterpret_cast<const f16x8*>(hi + at);
        in.lo = *reinterpret_cast<const u32x4*>(lo + at / 2);
        if (!tall) in.d = a + diagonal[i];
    }
    __device__ __forceinline__ void x(const In& in, float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float rest = as_f32(e & 1 ? in.lo[e / 2] & 0xffff0000u : in.lo[e / 2] << 16);
            v[e] = fmaf(tall ? d[e] : in.d, (float)in.hi[e] + rest, v[e]) * scale;
            rounded(v[e]);
        }
    }
};

struct ApplyOut : ApplyIn {
    static constexpr bool kColumns = true;
    _Float16 *next_hi, *next_t;
    __device__ __forceinline__ void row(int i, int j, const In& in, float (&v)[8]) const {
        if (i >= rows || j >= cols) return;
        x(in, v);
        const f16x8 h = half8(v);
        u32x4 low;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f32x2 rest = {v[2 * e] - (float)h[2 * e], v[2 * e + 1] - (float)h[2 * e + 1]};
            low[e] = __builtin_bit_cast(u32, __builtin_convertvector(rest, bf16x2));
        }
        const int64_t at = (int64_t)i * cols + j;
        *reinterpret_cast<f16x8*>(next_hi + at) = h;
        *reinterpret_cast<u32x4*>(lo + at / 2) = low;
    }
    __device__ __forceinline__ bool columns() const { return true; }
    __device__ __forceinline__ void column(int i, int j, const float (&v)[8]) const {
        if (i >= rows || j >= cols) return;
        *reinterpret_cast<f16x8*>(next_t + (int64_t)j * rows + i) = half8(v);
    }
};

// What the last step does with the result: hands it out as bfloat16, or moves the weights along it.
struct LastArgs {
    uint16_t* result;               // rows x cols matrices one after the other
    const fo_tensor_desc* matrices;
    float keep;                     // 1 - lr * weight decay
};

struct ResultOut : ApplyIn {
    static constexpr bool kColumns = false;
    uint16_t* result;
    int true_rows, true_cols;
    __device__ __forceinline__ ResultOut(const ApplyIn& in, const LastArgs& last, const MatrixGroup& m, int k)
        : ApplyIn(in), result(last.result + (int64_t)(m.first + k) * m.rows * m.cols), true_rows(m.rows), true_cols(m.cols) {}
    __device__ __forceinline__ void row(int i, int j, const In& in, float (&v)[8]) const {
        if (i >= true_rows || j >= true_cols) return;
        x(in, v);
        store_values<DT_BF16>(v, result + (int64_t)i * true_cols + j, true_cols - j);
    }
};

// Eight weights of a row, the first `valid` of them there:  p <- p * keep - lr * x  at master precision.
template <int DT, int ECCB> struct Weights {
    static constexpr int PB = DTypeInfo<DT>::bytes, EPL = DTypeInfo<DT>::epl, kParts = 8 / EPL;
    Pack<PB, EPL> p[kParts];
    Pack<ECCB, EPL> e[kParts];
    __device__ __forceinline__ void load(const void* param, const void* ecc, int64_t at, int valid) {
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            load_piece<PB, EPL>(p[k], (const char*)param + (at + k * EPL) * PB, valid - k * EPL);
            load_piece<ECCB, EPL>(e[k], (const char*)ecc + (at + k * EPL) * ECCB, valid - k * EPL);
        }
    }
    __device__ __forceinline__ void move(const float (&x)[8], float keep, float lr, void* param, void* ecc, int64_t at, int valid) const {
#pragma unroll
        for (int k = 0; k < kParts; ++k) {
            Pack<PB, EPL> narrow;
            Pack<ECCB, EPL> rest;
            float w[EPL];
#pragma unroll
            for (int q = 0; q < EPL; ++q) {
                float master = widen<DT, EPL>(p[k], q);
                if constexpr (ECCB > 0) master = ecc_join<DT, ECCB>(master, ecc_to_float<ECCB, EPL>(e[k], q));
                w[q] = master * keep - x[k * EPL + q] * lr;
            }
            write_master<DT, ECCB, EPL>(w, narrow, rest);
            store_piece<PB, EPL>(narrow, (char*)param + (at + k * EPL) * PB, valid - k * EPL);
            store_piece<ECCB, EPL>(rest, (char*)ecc + (at + k * EPL) * ECCB, valid - k * EPL);
        }
    }
};

template <int DT, int ECCB> struct UpdateOut : ApplyIn {
    static constexpr bool kColumns = false;
    void *param, *ecc;
    int true_rows, true_cols;
    float keep, lr;
    struct In : ApplyIn::In { Weights<DT, ECCB> w; };
    __device__ __forceinline__ UpdateOut(const ApplyIn& in, const LastArgs& last, const MatrixGroup& m, int k)
        : ApplyIn(in), true_rows(m.rows), true_cols(m.cols), keep(last.keep), lr(m.lr) {
        const fo_tensor_desc& d = last.matrices[m.first + k];
        param = d.param;
        ecc = d.ecc;
    }
    __device__ __forceinline__ void load(int i, int j, In& in) const {
        if (i >= true_rows || j >= true_cols) return;
        ApplyIn::load(i, j, in);
        in.w.load(param, ecc, (int64_t)i * true_cols + j, true_cols - j);
    }
    __device__ __forceinline__ void row(int i, int j, const In& in, float (&v)[8]) const {
        if (i >= true_rows || j >= true_cols) return;
        x(in, v);
        in.w.move(v, keep, lr, param, ecc, (int64_t)i * true_cols + j, true_cols - j);
    }
};

// Out: ApplyOut, or what the last step does.  14336 x 4096 in 533 us, 900 TFLOP/s (the median; 489 at least): a round of 256 x 256 tiles takes 135 us, 35 of which
// its epilogues' 10 bytes an element would take alone, and the card's clock falls under such products.
template <int WT, int STAGES, class Out> __global__ __launch_bounds__(256, WT >= 96 ? 1 : 2) void apply_kernel(Groups a, StepArgs h, LastArgs last) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    typedef GemmTile<F16Product, WT, STAGES> Tile;
    const int64_t seat = blockIdx.x >> 3;
    const int g = group_of(a, seat);
    const MatrixGroup& m = a.group[g];
    const int row_end = m.padded_rows < h.row_end ? m.padded_rows : h.row_end, col_end = m.padded_cols < h.col_end ? m.padded_cols : h.col_end;
    const int rows = (row_end - h.row_begin + Tile::kTile - 1) / Tile::kTile, cols = (col_end - h.col_begin + Tile::kTile - 1) / Tile::kTile;
    const int64_t local = tile_of_seat(blockIdx.x & 7, seat - a.begin[g], (int64_t)rows * cols * m.count);
    if (local < 0) return;
    const int k = (int)(local / (rows * cols));
    int i, j;
    tile_at((int)(local % (rows * cols)), rows, cols, i, j);
    const bool tall = m.tall();
    const int side = m.side();
    const Operand poly{(const char*)m.square(k, h.poly), side * 2, nullptr, 0, side};
    const Operand main{(const char*)m.hi(k, m.generation), side * 2, nullptr, 0, m.padded_rows};
    const Operand turned{(const char*)m.t(k, m.generation), side * 2, nullptr, 0, m.padded_cols};
    Tile tile(lds);
    const int row0 = h.row_begin + i * Tile::kTile, col0 = h.col_begin + j * Tile::kTile;
    tile.multiply(tall ? main : poly, tall ? poly : turned, row0, col0, side * 2);
    const ApplyIn in{m.hi(k, m.generation), m.lo(k), m.diagonal(k, h.poly), m.padded_rows, m.padded_cols, h.a, h.first ? 1.0f / m.unit : 1.0f, tall, {}};
    if constexpr (Out::kColumns) {
        Out out{in, m.hi(k, m.generation ^ 1), m.t(k, m.generation ^ 1)};
        tile.finish(row0, col0, out);
    } else {
        Out out(in, last, m, k);
        tile.finish(row0, col0, out);
    }
}

// ------------------------------------------------------------------------------------------------
// matrices that one workgroup holds
// ------------------------------------------------------------------------------------------------
// The whole iteration in one launch, a workgroup of 16 wavefronts per matrix: the fp32 X stays in registers in the layout the
// matrix instructions leave it in; LDS holds X's columns (T), S and B.  S is made of T through transposing LDS reads.  What bounds
// it is the chain of four phases per step with a barrier between them: 128 x 256 takes 39 us where a launch per product takes 81, 64 such
// matrices 44.
constexpr int kSmallThreads = 1024, kSmallWaves = kSmallThreads / 64;
constexpr int kSmallUnits = 4;                  // pieces of 32 x 16 of X per wavefront, side by side
constexpr int kSmallLds = 163840;
constexpr int kSmallPieces = 4;                 // 8-value pieces of G's rows per thread

// X is side x length, padded to multiples of 32.
struct SmallShape {
    int side, length;
    __host__ __device__ explicit SmallShape(const MatrixGroup& m) {
        side = ((m.tall() ? m.cols : m.rows) + 31) / 32 * 32;
        length = ((m.tall() ? m.rows : m.cols) + 31) / 32 * 32;
    }
    __host__ __device__ int pitch() const { return side * 2 + 16; }   // bytes; 16 rows' 16-byte pieces lie in different banks
    __host__ __device__ int gram() const { return length * pitch(); }   // where S begins; then B, then their diagonals
    __host__ __device__ int lds() const { return gram() + 2 * side * pitch() + 8 * side; }
    __host__ __device__ int waves_across() const { return (length + 16 * kSmallUnits - 1) / (16 * kSmallUnits); }
    // one 32 x 32 block of S per wavefront
    __host__ __device__ bool fits() const {
        const int blocks = side / 32;
        // (G itself, in fp32, takes 135168 bytes at most and four pieces per thread)
        // the counts first: beyond them lds() can pass 32 bits
        return blocks * waves_across() <= kSmallWaves && blocks * (blocks + 1) / 2 <= kSmallWaves && lds() <= kSmallLds;
    }
};

// A lane's places in a matrix in LDS: byte offsets that depend on the lane, to which the place of a block is added, the same
// for all lanes.
struct SmallPlaces {
    int pitch;
    int read_from;      // row `lane & 15`, columns (lane >> 4) * 8 on: an operand
    int turn_from;      // an operand of the transpose: in each 16 lanes, the columns of four rows, see read_turned
    int put_from[4];    // rows (lane >> 4) * 4 + e, column `lane & 15`: a result
    int put4_from;      // row `lane & 15`, columns (lane >> 4) * 4 on: a result transposed
    __device__ __forceinline__ SmallPlaces(int pitch, int lane) : pitch(pitch) {
        const int line = lane & 15, quad = (lane >> 4) * 4;
        read_from = line * pitch + quad * 4;
        turn_from = (quad * 2 + (line >> 2)) * pitch + (line & 3) * 8;
        put4_from = line * pitch + quad * 2;
#pragma unroll
        for (int e = 0; e < 4; ++e) put_from[e] = (quad + e) * pitch + line * 2;
    }
    __device__ __forceinline__ int block(int row, int col) const { return row * pitch + col * 2; }
};
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f16x8 read_piece(const char* lds, int at) { return *reinterpret_cast<const f16x8*>(lds + at); }
// Rows of the transpose: lane i of each 16 gives the address of four values and gets value i of what lanes 0..3, 4..7, 8..11 and
// 12..15 point at (16 values each).  Two such reads make an operand's eight values along k.
__device__ __forceinline__ f16x8 read_turned(char* lds, int at, int pitch) {
    typedef __attribute__((address_space(3))) s16x4* place;
    const f16x4 lo = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(lds + at)));
    const f16x4 hi = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((place)(lds + at + 4 * pitch)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ void put_half(char* lds, int at, _Float16 v) { *reinterpret_cast<_Float16*>(lds + at) = v; }
__device__ __forceinline__ void put_halves(char* lds, int at, f16x4 v) { *reinterpret_cast<f16x4*>(lds + at) = v; }
__device__ __forceinline__ f16x4 halves(f32x4 v) { return f16x4{(_Float16)v.x, (_Float16)v.y, (_Float16)v.z, (_Float16)v.w}; }

// What becomes of eight values of the result; what that needs from memory is loaded before the result is there.
struct SmallResult {
    uint16_t* result;
    struct In {};
    __device__ __forceinline__ SmallResult(const LastArgs& last, const MatrixGroup& m, int k) : result(last.result + (int64_t)(m.first + k) * m.rows * m.cols) {}
    __device__ __forceinline__ void load(int64_t, int, In&) const {}
    __device__ __forceinline__ void take(int64_t at, int valid, const float (&x)[8], const In&) const { store_values<DT_BF16>(x, result + at, valid); }
};
template <int DT, int ECCB> struct SmallUpdate {
    void *param, *ecc;
    float keep, lr;
    typedef Weights<DT, ECCB> In;
    __device__ __forceinline__ SmallUpdate(const LastArgs& last, const MatrixGroup& m, int k)
        : param(last.matrices[m.first + k].param), ecc(last.matrices[m.first + k].ecc), keep(last.keep), lr(m.lr) {}
    __device__ __forceinline__ void load(int64_t at, int valid, In& in) const { in.load(param, ecc, at, valid); }
    __device__ __forceinline__ void take(int64_t at, int valid, const float (&x)[8], const In& in) const { in.move(x, keep, lr, param, ecc, at, valid); }
};

// 32 x 32 block (bi, bj) of rows times rows over `length` values; TURNED: the rows are columns of what LDS holds.
template <bool TURNED> __device__ __forceinline__ void small_block(char* rows, const SmallPlaces& p, int bi, int bj, int length, f32x4 (&acc)[2][2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int a_from = TURNED ? p.turn_from + bi * 64 : p.read_from + p.block(bi * 32, 0);
    int b_from = TURNED ? p.turn_from + bj * 64 : p.read_from + p.block(bj * 32, 0);
    const int next_rows = TURNED ? 32 : p.block(16, 0), next_values = TURNED ? p.block(32, 0) : 64;
    for (int at = 0; at < length; at += 32) {
        f16x8 a[2], b[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            a[i] = TURNED ? read_turned(rows, a_from + i * next_rows, p.pitch) : read_piece(rows, a_from + i * next_rows);
            b[i] = TURNED ? read_turned(rows, b_from + i * next_rows, p.pitch) : read_piece(rows, b_from + i * next_rows);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i], b[j], acc[i][j], 0, 0, 0);
        a_from += next_values;
        b_from += next_values;
    }
}
// Puts block (bi, bj) of a symmetric matrix and its mirror image.
__device__ __forceinline__ void put_block(char* to, const SmallPlaces& p, int bi, int bj, const f16x4 (&v)[2][2]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = bi * 32 + i * 16, col = bj * 32 + j * 16;
            put_halves(to, p.put4_from + p.block(col, row), v[i][j]);
            if (bi != bj) {
#pragma unroll
                for (int e = 0; e < 4; ++e) put_half(to, p.put_from[e] + p.block(row, col), v[i][j][e]);
            }
        }
}

struct SmallArgs {
    float a, b, c, eps;
    int steps;
};

template <int DT, class Out> __global__ __launch_bounds__(kSmallThreads) void small_kernel(Groups groups, MatrixSource source, SmallArgs h, LastArgs last) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int g = group_of(groups, blockIdx.x);
    const MatrixGroup& m = groups.group[g];
    const int k = (int)(blockIdx.x - groups.begin[g]);
    const SmallShape shape(m);
    const int side = shape.side, length = shape.length;
    char *const t = lds, *const gram_rows = lds + shape.gram(), *const poly_rows = gram_rows + side * shape.pitch();
    float *const s_diagonal = reinterpret_cast<float*>(poly_rows + side * shape.pitch()), *const diagonal = s_diagonal + side;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int line = lane & 15, quad = (lane >> 4) * 4;

    // The wavefront's pieces of X.  Where there are fewer than places for them, places share a piece: they work out and
    // write the same values, and nothing below asks.
    const int across = shape.waves_across(), whole_waves = side / 32 * across, mine = wave < whole_waves ? wave : whole_waves - 1;
    const int row_of = mine / across * 32;
    int col_of[kSmallUnits];
#pragma unroll
    for (int u = 0; u < kSmallUnits; ++u) {
        const int col = mine % across * 16 * kSmallUnits + u * 16;
        col_of[u] = col < length ? col : length - 16;
    }
    const bool tall = m.tall();
    const char* in = source.data ? (const char*)source.data + source.stride * k * DTypeInfo<DT>::bytes : (const char*)m.update(k);
    const int64_t row_stride = source.data ? source.row_stride : m.cols;
    // G passes through LDS in fp32, row by row in 8-value pieces here, as the instructions lay X out there
    float* const whole = reinterpret_cast<float*>(lds);
    const int pitch = m.cols | 1, row_step = tall ? 1 : pitch, col_step = tall ? pitch : 1;
    const int pieces = (m.cols + 7) / 8, all = pieces * m.rows;
    double total;
    {
        float v[kSmallPieces][8], quick = 0.0f;
#pragma unroll
        for (int i = 0; i < kSmallPieces; ++i) {
            const int at = threadIdx.x + i * kSmallThreads, row = at / pieces, col = (at - row * pieces) * 8;
            if (at < all) read8<DT>(in + (row_stride * row + col) * DTypeInfo<DT>::bytes, m.cols - col, v[i]);
        }
#pragma unroll
        for (int i = 0; i < kSmallPieces; ++i) {
            const int at = threadIdx.x + i * kSmallThreads, row = at / pieces, col = (at - row * pieces) * 8;
            if (at < all) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (col + e < m.cols) whole[row * pitch + col + e] = v[i][e];
                    quick = fmaf(v[i][e], v[i][e], quick);
                }
            }
        }
        total = (double)quick;
        if (!holds_squares(quick)) {
            total = 0.0;
#pragma unroll
            for (int i = 0; i < kSmallPieces; ++i)
                if ((int)threadIdx.x + i * kSmallThreads < all) total += sum_of_squares(v[i]);
        }
    }
    __syncthreads();
    const int true_side = tall ? m.cols : m.rows, true_length = tall ? m.rows : m.cols;
    f32x4 x[kSmallUnits][2];
#pragma unroll
    for (int u = 0; u < kSmallUnits; ++u) {
        const int row = row_of + quad, col = col_of[u] + line;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool there = row + half * 16 + e < true_side && col < true_length;
                const float v = whole[there ? (row + half * 16 + e) * row_step + col * col_step : 0];
                x[u][half][e] = there ? v : 0.0f;
            }
    }
    __syncthreads();
    double* sums = reinterpret_cast<double*>(lds);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) total += __shfl_down(total, d);
    if (lane == 0) sums[wave] = total;
    __syncthreads();
    total = 0.0;
#pragma unroll
    for (int w = 0; w < kSmallWaves; ++w) total += sums[w];
    double norm = sqrt(total) + (double)h.eps;
    __syncthreads();
    const float power = power_for(norm);
    if (power != 1.0f) {   // seldom
        norm *= (double)power;
#pragma unroll
        for (int u = 0; u < kSmallUnits; ++u) { x[u][0] *= power; x[u][1] *= power; }
    }
    const float factor = (float)(1.0 / norm);
#pragma unroll
    for (int u = 0; u < kSmallUnits; ++u) { x[u][0] *= factor; x[u][1] *= factor; }

    // the wavefront's block of S and B, on or above the diagonal, column by column
    int bi = wave, bj = 0;
    while (bi > bj) { ++bj; bi -= bj; }
    const bool has_block = bj < side / 32;
    const SmallPlaces at(shape.pitch(), lane);
    for (int step = 0; step < h.steps; ++step) {
#pragma unroll
        for (int u = 0; u < kSmallUnits; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) put_halves(t, at.put4_from + at.block(col_of[u], row_of + half * 16), halves(x[u][half]));
        __syncthreads();
        f32x4 gram[2][2];
        if (has_block) {
            f16x4 v[2][2];
            small_block<true>(t, at, bi, bj, length, gram);
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (bi == bj && p == q && quad + e == line) { s_diagonal[bi * 32 + p * 16 + line] = gram[p][q][e]; gram[p][q][e] = 0.0f; }
                    v[p][q] = halves(gram[p][q]);
                    // B is made of S as the products see it: its two terms nearly cancel near the end of the iteration
#pragma unroll
                    for (int e = 0; e < 4; ++e) gram[p][q][e] = (float)v[p][q][e];
                }
            put_block(gram_rows, at, bi, bj, v);
        }
        __syncthreads();
        if (has_block) {
            f32x4 squared[2][2];
            f16x4 w[2][2];
            small_block<false>(gram_rows, at, bi, bj, side, squared);
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const f32x4 di = *reinterpret_cast<const f32x4*>(s_diagonal + bi * 32 + p * 16 + quad);
                    const float dj = s_diagonal[bj * 32 + q * 16 + line];
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = fmaf(h.c, fmaf(di[e] + dj, gram[p][q][e], squared[p][q][e]), h.b * gram[p][q][e]);
                        if (bi == bj && p == q && quad + e == line) { diagonal[bi * 32 + p * 16 + line] = fmaf(dj, fmaf(h.c, dj, h.b), v[e]); v[e] = 0.0f; }
                    }
                    w[p][q] = halves(v);
                }
            put_block(poly_rows, at, bi, bj, w);
        }
        __syncthreads();
        f32x4 acc[kSmallUnits][2];
#pragma unroll
        for (int u = 0; u < kSmallUnits; ++u) acc[u][0] = acc[u][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int from = 0; from < side; from += 32) {
            const f16x8 poly0 = read_piece(poly_rows, at.read_from + at.block(row_of, from)), poly1 = read_piece(poly_rows, at.read_from + at.block(row_of + 16, from));
#pragma unroll
            for (int u = 0; u < kSmallUnits; ++u) {
                const f16x8 column = read_piece(t, at.read_from + at.block(col_of[u], from));
                acc[u][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(poly0, column, acc[u][0], 0, 0, 0);
                acc[u][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(poly1, column, acc[u][1], 0, 0, 0);
            }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const f32x4 d = *reinterpret_cast<const f32x4*>(diagonal + row_of + quad + half * 16);
#pragma unroll
            for (int u = 0; u < kSmallUnits; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][half][e] = fmaf(h.a + d[e], x[u][half][e], acc[u][half][e]);
        }
        __syncthreads();
    }
    // places worked out again, not kept from the beginning
    int thread = threadIdx.x, last_line = line, last_quad = quad;
    asm volatile("" : "+v"(thread), "+v"(last_line), "+v"(last_quad));
    const Out out(last, m, k);
    typename Out::In with[kSmallPieces];
#pragma unroll
    for (int i = 0; i < kSmallPieces; ++i) {
        const int at = thread + i * kSmallThreads, row = at / pieces, col = (at - row * pieces) * 8;
        if (at < all) out.load((int64_t)row * m.cols + col, m.cols - col, with[i]);
    }
#pragma unroll
    for (int u = 0; u < kSmallUnits; ++u) {
        const int row = row_of + last_quad, col = col_of[u] + last_line;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (row + half * 16 + e < true_side && col < true_length) whole[(row + half * 16 + e) * row_step + col * col_step] = x[u][half][e];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSmallPieces; ++i) {
        const int at = thread + i * kSmallThreads, row = at / pieces, col = (at - row * pieces) * 8;
        if (at >= all) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = whole[row * pitch + (col + e < m.cols ? col + e : 0)];
        out.take((int64_t)row * m.cols + col, m.cols - col, v, with[i]);
    }
}

// ------------------------------------------------------------------------------------------------
// matrices that one wavefront holds
// ------------------------------------------------------------------------------------------------
// Sixteen rows of up to 64 values at most: a lane has a column of X in registers, S and B lie in LDS, and all of it is fp32 on the
// vector units.  Not for speed: where the sides are this short a matrix is often nearly singular, and then the roundings to
// fp16 above, which longer sides average out, reach 1e-2 of the result (4000 random matrices of each shape: 4e-2 at 2 x 2, 7e-3 at 8 x 8,
// 1.8e-3 at 8 x 32; above these sizes 1.3e-3 at most).  8 x 8 takes 15 us, 4096 of 16 x 16 take 29.
constexpr int kTinySide = 16, kTinyLength = 64, kTinyPieces = 2;   // 8-value pieces of G's rows per lane

template <int DT, class Out> __global__ __launch_bounds__(64) void tiny_kernel(Groups groups, MatrixSource source, SmallArgs h, LastArgs last) {
    __shared__ float xs[kTinySide][kTinyLength + 1];
    __shared__ __attribute__((aligned(16))) float s[kTinySide][kTinySide + 4], b[kTinySide][kTinySide + 4];
    const int g = group_of(groups, blockIdx.x);
    const MatrixGroup& m = groups.group[g];
    const int k = (int)(blockIdx.x - groups.begin[g]), lane = threadIdx.x;
    const bool tall = m.tall();
    const int length = tall ? m.rows : m.cols, pieces = (m.cols + 7) / 8, all = pieces * m.rows;
    const char* in = source.data ? (const char*)source.data + source.stride * k * DTypeInfo<DT>::bytes : (const char*)m.update(k);
    const int64_t row_stride = source.data ? source.row_stride : m.cols;
    const Out out(last, m, k);
    typename Out::In with[kTinyPieces];
    float x[kTinySide];
#pragma unroll
    for (int i = 0; i < kTinySide; ++i) xs[i][lane] = 0.0f;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTinyPieces; ++i) {
        const int at = lane + i * 64, row = at / pieces, col = (at - row * pieces) * 8;
        if (at >= all) continue;
        float v[8];
        read8<DT>(in + (row_stride * row + col) * DTypeInfo<DT>::bytes, m.cols - col, v);
        out.load((int64_t)row * m.cols + col, m.cols - col, with[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (col + e < m.cols) xs[tall ? col + e : row][tall ? row : col + e] = v[e];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTinySide; ++i) x[i] = xs[i][lane];
    double total = sum_of_squares(x);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) total += __shfl_xor(total, d);
    const double norm = sqrt(total) + (double)h.eps;
    const float power = power_for(norm), factor = (float)(1.0 / (norm * (double)power));
#pragma unroll
    for (int i = 0; i < kTinySide; ++i) x[i] = x[i] * power * factor;
    const int row = lane >> 2, first = (lane & 3) * 4;   // the lane's four entries of S and B
    for (int step = 0; step < h.steps; ++step) {
#pragma unroll
        for (int i = 0; i < kTinySide; ++i) xs[i][lane] = x[i];
        __syncthreads();
        float gram[4] = {0.0f, 0.0f, 0.0f, 0.0f}, squared[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int c = 0; c < length; ++c) {
            const float v = xs[row][c];
#pragma unroll
            for (int e = 0; e < 4; ++e) gram[e] = fmaf(v, xs[first + e][c], gram[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[row][first + e] = gram[e];
        __syncthreads();
#pragma unroll
        for (int c = 0; c < kTinySide; ++c) {
            const float v = s[row][c];
#pragma unroll
            for (int e = 0; e < 4; ++e) squared[e] = fmaf(v, s[c][first + e], squared[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) b[row][first + e] = fmaf(h.c, squared[e], h.b * gram[e]);
        __syncthreads();
        float next[kTinySide];
#pragma unroll
        for (int i = 0; i < kTinySide; ++i) {
            next[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < kTinySide; ++j) next[i] = fmaf(b[i][j], x[j], next[i]);
        }
#pragma unroll
        for (int i = 0; i < kTinySide; ++i) x[i] = fmaf(h.a, x[i], next[i]);
    }
#pragma unroll
    for (int i = 0; i < kTinySide; ++i) xs[i][lane] = x[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTinyPieces; ++i) {
        const int at = lane + i * 64, row = at / pieces, col = (at - row * pieces) * 8;
        if (at >= all) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = col + e < m.cols ? xs[tall ? col + e : row][tall ? row : col + e] : 0.0f;
        out.take((int64_t)row * m.cols + col, m.cols - col, v, with[i]);
    }
}

}  // namespace fo

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
namespace {
using namespace fo_host;

constexpr int64_t kMostWorkgroups = 1 << 21;   // of up to 1024 threads: below 2^32 work-items

int padded(int n, bool shorter) { return shorter && n <= fo::kNarrow ? fo::kNarrow : (n + fo::kPad - 1) / fo::kPad * fo::kPad; }

// Shapes without elements are left out of the launches.
int validate_shapes(const fo_matrix_shape* shapes, int64_t n) {
    if (n < 0 || (n > 0 && !shapes)) return fail(FO_ERR_INVALID_ARGUMENT, "shapes must not be NULL");
    for (int64_t i = 0; i < n; ++i) {
        const fo_matrix_shape& s = shapes[i];
        if (s.rows < 0 || s.cols < 0 || s.count < 0) return fail(FO_ERR_INVALID_ARGUMENT, "negative size of shape %lld", (long long)i);
        if (s.rows > FO_MATRIX_MOST_LINES || s.cols > FO_MATRIX_MOST_LINES)
            return fail(FO_ERR_UNSUPPORTED, "a matrix of %d x %d has more than %d rows or columns", s.rows, s.cols, FO_MATRIX_MOST_LINES);
    }
    return 0;
}

// The groups of shapes[0..n) with their places in the workspace; returns its size.
int64_t plan(const fo_matrix_shape* shapes, int64_t n, char* workspace, fo::Groups* out) {
    int64_t at = 0;
    int first = 0, used = 0;
    for (int64_t i = 0; i < n; ++i) {
        const fo_matrix_shape& s = shapes[i];
        if (s.rows > 0 && s.cols > 0 && s.count > 0) {
            fo::MatrixGroup m{};
            m.rows = s.rows; m.cols = s.cols; m.count = s.count; m.first = first; m.lr = s.lr;
            m.padded_rows = padded(s.rows, s.rows <= s.cols); m.padded_cols = padded(s.cols, s.rows > s.cols);
            m.chunks = (int)(((int64_t)s.rows * s.cols + fo::kChunk - 1) / fo::kChunk);
            m.unit = 1.0f;
            m.parts = 1;
            const int longer = s.rows > s.cols ? s.rows : s.cols;
            while (m.unit * m.unit * 4.0f <= (float)longer) m.unit *= 2.0f;
            m.workspace = workspace + at;
            at += m.bytes_each() * s.count;
            if (out) out->group[used] = m;
            ++used;
        }
        first += s.count;
    }
    if (out) {
        out->n = used;
        // the longest contractions first: what is left at the end of a launch is short
        std::stable_sort(out->group, out->group + used, [](const fo::MatrixGroup& x, const fo::MatrixGroup& y) {
            return std::max(x.rows, x.cols) > std::max(y.rows, y.cols);
        });
    }
    return at;
}

// Sets the groups' ranges of workgroups, `each(group)` of them for a matrix; returns the grid.
template <class F> int64_t spread(fo::Groups& a, F each) {
    a.begin[0] = 0;
    for (int g = 0; g < a.n; ++g) a.begin[g + 1] = a.begin[g] + each(a.group[g]) * a.group[g].count;
    return a.begin[a.n];
}

// The groups that `which` picks, a workgroup to a matrix; with `leave` they are gone from `a`.
fo::Groups take(fo::Groups& a, bool (*which)(const fo::MatrixGroup&), bool leave) {
    fo::Groups taken{}, left{};
    for (int g = 0; g < a.n; ++g) {
        fo::Groups& to = which(a.group[g]) ? taken : left;
        to.group[to.n++] = a.group[g];
    }
    if (leave) a = left;
    spread(taken, [](const fo::MatrixGroup&) { return (int64_t)1; });
    return taken;
}

int64_t tiles_across(int n, int tile) { return (n + tile - 1) / tile; }

template <class K, class... Args> int launch(K kernel, int64_t grid, int threads, int lds, hipStream_t stream, const char* what, Args... args) {
    if (grid > kMostWorkgroups) return fail(FO_ERR_UNSUPPORTED, "%s: %lld workgroups are more than one launch takes", what, (long long)grid);
    if (lds > 65536) {
        if (int rc = check_hip(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds), what)) return rc;
    }
    kernel<<<dim3((unsigned)grid), dim3(threads), lds, stream>>>(args...);
    return check_hip(hipGetLastError(), what);
}

// Which tile a launch takes: the one whose rounds over the compute units take least, by times fitted to steps of 4096 x 14336, 4096 x
// 4096, 1024 x 4096 and 1000 x 2730 matrices: 131 us for a 256 x 256 tile over 4096 values, 80 for 192 x 192, 75 for two
// 128 x 128, 52 for five 64 x 64 (the smaller ones read more of LDS per multiplication); 43, 33, 24 (21 alone) and 18 (11) over 1024.
constexpr fo::TileCost kTileCosts[] = {
    {128, 2, 1, 14.0, 0.0286, 14.0, 0.0286}, {96, 3, 1, 19.0, 0.0150, 19.0, 0.0150}, {64, 2, 2, 9.5, 0.0115, 8.0, 0.0165},
    {32, 2, 5, 4.2, 0.0063, 7.0, 0.0110}, {32, 4, 2, 4.2, 0.0036, 7.0, 0.0058}};

// tiles(group, wt) of a matrix, length(group) contracted.
template <class T, class L> fo::TileCost choose(const fo::Groups& a, int cus, T tiles, L length, double& least) {
    fo::TileCost best{};
    least = 0.0;
    for (const fo::TileCost& t : kTileCosts) {
        double all = 0.0, values = 0.0;
        for (int g = 0; g < a.n; ++g) {
            const double n = (double)tiles(a.group[g], t.wt) * a.group[g].count;
            all += n;
            values += n * length(a.group[g]);
        }
        const double time = fo::tiles_time(t, all, values / all, cus);
        if (!best.wt || time < least) { best = t; least = time; }
    }
    return best;
}

int64_t symmetric_tiles(const fo::MatrixGroup& m, int wt) { const int64_t n = tiles_across(m.side(), 2 * wt); return n * (n + 1) / 2; }
int64_t apply_tiles(const fo::MatrixGroup& m, int wt) { return fo::tiles_of(m.padded_rows, m.padded_cols, wt); }

// Seats per die, and the grid.
template <class F> int64_t seat(fo::Groups& a, F tiles) {
    a.begin[0] = 0;
    for (int g = 0; g < a.n; ++g) a.begin[g + 1] = a.begin[g] + fo::seats_of(tiles(a.group[g]) * a.group[g].count);
    return a.begin[a.n] * 8;
}

template <int WT, int STAGES, int KIND> int launch_symmetric(fo::Groups& a, const fo::SquareArgs& h, hipStream_t stream) {
    const int64_t grid = seat(a, [](const fo::MatrixGroup& m) { return symmetric_tiles(m, WT) * (KIND == fo::kPartial ? m.parts : 1); });
    return launch(fo::symmetric_kernel<WT, STAGES, KIND>, grid, 256, fo::GemmTile<fo::F16Product, WT, STAGES>::kLds, stream, "Newton-Schulz product", a, h);
}
template <int KIND> int launch_symmetric(const fo::TileCost& t, fo::Groups& a, const fo::SquareArgs& h, hipStream_t stream) {
    switch (t.wt) {
        case 128: return launch_symmetric<128, 2, KIND>(a, h, stream);
        case 96: return launch_symmetric<96, 3, KIND>(a, h, stream);
        case 64: return launch_symmetric<64, 2, KIND>(a, h, stream);
        default: return t.stages == 4 ? launch_symmetric<32, 4, KIND>(a, h, stream) : launch_symmetric<32, 2, KIND>(a, h, stream);
    }
}
template <int KIND> int launch_square(fo::Groups& a, const fo::SquareArgs& h, int cus, hipStream_t stream) {
    double least;
    return launch_symmetric<KIND>(choose(a, cus, symmetric_tiles, [](const fo::MatrixGroup& m) { return m.side(); }, least), a, h, stream);
}

int long_axis(const fo::MatrixGroup& m) { return m.tall() ? m.padded_rows : m.padded_cols; }
constexpr int kPartialMost = 64;   // few and short parts are what small tiles are for
// At most `most`, of whole stages of 64 values, none of them empty.
int parts_of(const fo::MatrixGroup& m, int most) {
    const int stages = long_axis(m) / 64, parts = std::max(1, std::min({most, m.most_parts(), stages / 2})), run = (stages + parts - 1) / parts;
    return (stages + run - 1) / run;
}

// S has few tiles where one side is short, each contracted over the whole other side.  Then the long axis is cut into parts that
// are contracted at the same time and added up: 64 x 14336 takes 115 instead of 249 us in all, 300 x 9000 154 instead of 222,
// 1024 x 14336 486 instead of 499.
// How many parts goes by the shape alone, so that a matrix's result does not depend on what shares the launch; a tenth of the time has
// to be gained by it.
int gram_parts(const fo::MatrixGroup& m, int cus) {
    double least = 0.0;
    int best = 1;
    for (const fo::TileCost& t : kTileCosts) {
        const double time = 0.9 * fo::tiles_time(t, (double)symmetric_tiles(m, t.wt), long_axis(m), cus);
        if (least == 0.0 || time < least) least = time;
    }
    for (int most = 2; most <= 128; most *= 2) {
        for (const fo::TileCost& t : kTileCosts) {
            if (t.wt > kPartialMost) continue;
            const int parts = parts_of(m, most);
            const double time = fo::tiles_time(t, (double)symmetric_tiles(m, t.wt) * parts, (double)long_axis(m) / parts, cus) + fo::kLaunchTime
                              + (double)m.gram_area() * parts * 1e-6 + 0.06 * parts;   // sums written and read, a row of loads of each
            if (time < least) { least = time; best = parts; }
        }
    }
    return best;
}
int launch_gram(fo::Groups& a, const fo::SquareArgs& h, int cus, hipStream_t stream) {
    fo::Groups parted = take(a, [](const fo::MatrixGroup& m) { return m.parts > 1; }, false), whole = take(a, [](const fo::MatrixGroup& m) { return m.parts == 1; }, false);
    double least;
    if (whole.n > 0) {
        const fo::TileCost t = choose(whole, cus, symmetric_tiles, long_axis, least);
        if (int rc = launch_symmetric<fo::kGram>(t, whole, h, stream)) return rc;
    }
    if (parted.n == 0) return 0;
    const fo::TileCost t = choose(parted, cus, [](const fo::MatrixGroup& m, int wt) { return symmetric_tiles(m, wt) * m.parts; },
                                  [](const fo::MatrixGroup& m) { return long_axis(m) / m.parts; }, least);
    if (int rc = t.wt >= kPartialMost ? launch_symmetric<kPartialMost, 2, fo::kPartial>(parted, h, stream)
               : t.stages == 4 ? launch_symmetric<32, 4, fo::kPartial>(parted, h, stream) : launch_symmetric<32, 2, fo::kPartial>(parted, h, stream)) return rc;
    const int64_t grid = spread(parted, [](const fo::MatrixGroup& m) { return symmetric_tiles(m, 32) * 16; });
    return launch(fo::gather_kernel, grid, 256, 0, stream, "Newton-Schulz sums", parted, h);
}
template <int WT, int STAGES, class Out> int launch_apply(fo::Groups& a, const fo::StepArgs& h, const fo::LastArgs& last, hipStream_t stream) {
    const int64_t grid = seat(a, [&](const fo::MatrixGroup& m) {
        return fo::tiles_of(std::min(m.padded_rows, h.row_end) - h.row_begin, std::min(m.padded_cols, h.col_end) - h.col_begin, WT);
    });
    return launch(fo::apply_kernel<WT, STAGES, Out>, grid, 256, fo::GemmTile<fo::F16Product, WT, STAGES>::kLds, stream, "Newton-Schulz step", a, h, last);
}
template <class Out> int launch_apply(const fo::TileCost& t, fo::Groups& a, const fo::StepArgs& h, const fo::LastArgs& last, hipStream_t stream) {
    switch (t.wt) {
        case 128: return launch_apply<128, 2, Out>(a, h, last, stream);
        case 96: return launch_apply<96, 3, Out>(a, h, last, stream);
        case 64: return launch_apply<64, 2, Out>(a, h, last, stream);
        default: return t.stages == 4 ? launch_apply<32, 4, Out>(a, h, last, stream) : launch_apply<32, 2, Out>(a, h, last, stream);
    }
}
// One matrix may be cut (fo_gemm.h); of several the rounds run on from one to the next.
template <class Out> int launch_apply(fo::Groups& a, const fo::StepArgs& h, const fo::LastArgs& last, int cus, hipStream_t stream) {
    const fo::MatrixGroup& m = a.group[0];
    double least;
    if (a.n > 1 || m.count > 1) return launch_apply<Out>(choose(a, cus, apply_tiles, [](const fo::MatrixGroup& m) { return m.side(); }, least), a, h, last, stream);
    const fo::Cut cut = fo::best_cut(kTileCosts, m.padded_rows, m.padded_cols, m.side(), [](int) { return 0.0; }, 0.0, cus);
    if (!cut.rest.wt) return launch_apply<Out>(cut.tile, a, h, last, stream);
    fo::StepArgs first = h, rest = h;
    if (cut.columns) first.col_end = rest.col_begin = cut.lines * 2 * cut.tile.wt;
    else first.row_end = rest.row_begin = cut.lines * 2 * cut.tile.wt;
    if (int rc = launch_apply<Out>(cut.tile, a, first, last, stream)) return rc;
    return launch_apply<Out>(cut.rest, a, rest, last, stream);
}
int launch_update(fo::Groups& a, const fo::StepArgs& h, const fo::LastArgs& last, int dtype, int ecc_bytes, int cus, hipStream_t stream) {
    if (dtype == FO_F32) return launch_apply<fo::UpdateOut<fo::DT_F32, 0>>(a, h, last, cus, stream);
    if (dtype == FO_BF16) return ecc_bytes == 0 ? launch_apply<fo::UpdateOut<fo::DT_BF16, 0>>(a, h, last, cus, stream)
                               : ecc_bytes == 1 ? launch_apply<fo::UpdateOut<fo::DT_BF16, 1>>(a, h, last, cus, stream)
                                                : launch_apply<fo::UpdateOut<fo::DT_BF16, 2>>(a, h, last, cus, stream);
    return ecc_bytes == 0 ? launch_apply<fo::UpdateOut<fo::DT_F16, 0>>(a, h, last, cus, stream)
         : ecc_bytes == 1 ? launch_apply<fo::UpdateOut<fo::DT_F16, 1>>(a, h, last, cus, stream)
                          : launch_apply<fo::UpdateOut<fo::DT_F16, 2>>(a, h, last, cus, stream);
}

struct Iteration { int steps; float a, b, c, eps; };

int validate_iteration(int steps, const float* coefficients, float eps) {
    if (steps < 1) return fail(FO_ERR_INVALID_ARGUMENT, "steps must be at least 1, not %d", steps);
    if (!coefficients) return fail(FO_ERR_INVALID_ARGUMENT, "coefficients must not be NULL");
    if (!(eps >= 0.0f)) return fail(FO_ERR_INVALID_ARGUMENT, "eps must not be negative");
    return 0;
}

// The shapes that one wavefront or one workgroup holds leave `a` and are done in a launch of their own.
bool is_tiny(const fo::MatrixGroup& m) { return std::min(m.rows, m.cols) <= fo::kTinySide && std::max(m.rows, m.cols) <= fo::kTinyLength; }
bool is_small(const fo::MatrixGroup& m) { return fo::SmallShape(m).fits(); }

template <int DT, class Out> int launch_held(fo::Groups& a, const fo::MatrixSource& source, const Iteration& it, const fo::LastArgs& last, hipStream_t stream) {
    const fo::SmallArgs h{it.a, it.b, it.c, it.eps, it.steps};
    const fo::Groups tiny = take(a, is_tiny, true);
    if (tiny.n > 0) {
        if (int rc = launch(fo::tiny_kernel<DT, Out>, tiny.begin[tiny.n], 64, 0, stream, "Newton-Schulz of the smallest matrices", tiny, source, h, last)) return rc;
    }
    const fo::Groups small = take(a, is_small, true);
    if (small.n == 0) return 0;
    return launch(fo::small_kernel<DT, Out>, small.begin[small.n], fo::kSmallThreads, fo::kSmallLds, stream, "Newton-Schulz of small matrices", small, source, h, last);
}
int launch_held_update(fo::Groups& a, const Iteration& it, const fo::LastArgs& last, int dtype, int ecc_bytes, hipStream_t stream) {
    const fo::MatrixSource s{nullptr, 0, 0};
    if (dtype == FO_F32) return launch_held<fo::DT_F32, fo::SmallUpdate<fo::DT_F32, 0>>(a, s, it, last, stream);
    if (dtype == FO_BF16) return ecc_bytes == 0 ? launch_held<fo::DT_F32, fo::SmallUpdate<fo::DT_BF16, 0>>(a, s, it, last, stream)
                               : ecc_bytes == 1 ? launch_held<fo::DT_F32, fo::SmallUpdate<fo::DT_BF16, 1>>(a, s, it, last, stream)
                                                : launch_held<fo::DT_F32, fo::SmallUpdate<fo::DT_BF16, 2>>(a, s, it, last, stream);
    return ecc_bytes == 0 ? launch_held<fo::DT_F32, fo::SmallUpdate<fo::DT_F16, 0>>(a, s, it, last, stream)
         : ecc_bytes == 1 ? launch_held<fo::DT_F32, fo::SmallUpdate<fo::DT_F16, 1>>(a, s, it, last, stream)
                          : launch_held<fo::DT_F32, fo::SmallUpdate<fo::DT_F16, 2>>(a, s, it, last, stream);
}

// The products of one or two steps over the matrices of `a`.
struct Steps {
    const Iteration& it;
    int cus;
    hipStream_t stream;

    int gram(fo::Groups& a, int out, int first) const { return launch_gram(a, fo::SquareArgs{0, 0, out, 0.0f, 0.0f, 0.0f, first}, cus, stream); }
    int square(fo::Groups& a, int u, int v, int out, float alpha, float beta, float gamma) const {
        return launch_square<fo::kMixed>(a, fo::SquareArgs{u, v, out, alpha, beta, gamma, 0}, cus, stream);
    }
    // B of S
    int poly(fo::Groups& a, int s, int out) const { return launch_square<fo::kPoly>(a, fo::SquareArgs{s, s, out, it.b, 0.0f, it.c, 0}, cus, stream); }

    // Up to X's own product.
    int one(fo::Groups& a, int first, fo::StepArgs& then) const {
        if (int rc = gram(a, 0, first)) return rc;
        if (int rc = poly(a, 0, 1)) return rc;
        then = fo::StepArgs{it.a, 1, first};
        return 0;
    }
    // The first two: B1 of S, T = (a + B1) S, S2 = T (a + B1), B2 of it, and (a + B2) (a + B1) = a a + B2 B1 + a B2 + a B1.
    int two(fo::Groups& a, fo::StepArgs& then) const {
        if (int rc = gram(a, 0, 1)) return rc;
        if (int rc = poly(a, 0, 1)) return rc;
        if (int rc = square(a, 1, 0, 2, 0.0f, it.a, 1.0f)) return rc;
        if (int rc = square(a, 2, 1, 0, it.a, 0.0f, 1.0f)) return rc;
        if (int rc = poly(a, 0, 2)) return rc;
        if (int rc = square(a, 2, 1, 0, it.a, it.a, 1.0f)) return rc;
        then = fo::StepArgs{it.a * it.a, 0, 1};
        return 0;
    }
    // X's own product; finish(a, then) where it is the last.
    template <class F> int apply(fo::Groups& a, const fo::StepArgs& then, bool last, F finish) const {
        if (int rc = last ? finish(a, then, cus) : launch_apply<fo::ApplyOut>(a, then, fo::LastArgs{}, cus, stream)) return rc;
        for (int g = 0; g < a.n; ++g) a.group[g].generation ^= 1;
        return 0;
    }
};

// Whether the first two steps are merged.  14336 x 4096: 3.95 ms in all become 3.48; 512 x 14336: 255 us become 236, 512 x 4096: 170 become 161;
// 900 x 1800 takes 172 either way, 250 x 1000 115 and not 112, 1500 x 1000 174 and not 171; square matrices would only pay for it.
bool merges(const fo::MatrixGroup& m) { return 2 * std::max(m.rows, m.cols) >= 3 * std::min(m.rows, m.cols); }

// From the sums of squares on.  finish(a, step, cus) launches the last step.
template <int DT, class F> int iterate(fo::Groups& a, const fo::MatrixSource& source, const Iteration& it, hipStream_t stream, F finish) {
    const int cus = compute_units();
    if (cus <= 0) return fail(FO_ERR_NO_DEVICE, "no device");
    int64_t grid = spread(a, [](const fo::MatrixGroup&) { return (int64_t)1; });
    if (int rc = launch(fo::norm_kernel, grid, 256, 0, stream, "norm", a, it.eps)) return rc;
    grid = spread(a, [](const fo::MatrixGroup& m) { return fo::tiles_of(m.padded_rows, m.padded_cols, 32); });
    if (int rc = launch(fo::split_kernel<DT>, grid, 256, 0, stream, "normalisation", a, source)) return rc;
    for (int g = 0; g < a.n; ++g) a.group[g].parts = gram_parts(a.group[g], cus);
    const Steps steps{it, cus, stream};
    fo::StepArgs then{};
    int done = 0;
    if (it.steps >= 2) {
        fo::Groups merged{}, single{};
        for (int g = 0; g < a.n; ++g) {
            fo::Groups& to = merges(a.group[g]) ? merged : single;
            to.group[to.n++] = a.group[g];
        }
        if (merged.n > 0) {
            const bool last = it.steps == 2;
            if (int rc = steps.two(merged, then)) return rc;
            if (int rc = steps.apply(merged, then, last, finish)) return rc;
            for (int k = 0; k < 2 && single.n > 0; ++k) {
                if (int rc = steps.one(single, k == 0, then)) return rc;
                if (int rc = steps.apply(single, then, last && k == 1, finish)) return rc;
            }
            for (int g = 0, i = 0, j = 0; g < a.n; ++g) a.group[g] = merges(a.group[g]) ? merged.group[i++] : single.group[j++];
            done = 2;
        }
    }
    for (int k = done; k < it.steps; ++k) {
        if (int rc = steps.one(a, k == 0, then)) return rc;
        if (int rc = steps.apply(a, then, k + 1 == it.steps, finish)) return rc;
    }
    return 0;
}

template <int DT> int orthogonalise(fo::Groups& a, const fo::MatrixSource& source, const Iteration& it, const fo::LastArgs& last, hipStream_t stream) {
    if (int rc = launch_held<DT, fo::SmallResult>(a, source, it, last, stream)) return rc;
    if (a.n == 0) return 0;
    const int64_t grid = spread(a, [](const fo::MatrixGroup& m) { return (int64_t)m.chunks; });
    if (int rc = launch(fo::squares_kernel<DT>, grid, 256, 0, stream, "sum of squares", a, source)) return rc;
    return iterate<DT>(a, source, it, stream, [&](fo::Groups& some, const fo::StepArgs& h, int cus) { return launch_apply<fo::ResultOut>(some, h, last, cus, stream); });
}

template <int DT> int momentum(fo::Groups& a, const fo::MomentumArgs& h, int quantized, hipStream_t stream) {
    const int64_t grid = spread(a, [](const fo::MatrixGroup& m) { return (int64_t)m.chunks; });
    return quantized ? launch(fo::momentum_kernel<DT, true>, grid, 256, 0, stream, "momentum", a, h)
                     : launch(fo::momentum_kernel<DT, false>, grid, 256, 0, stream, "momentum", a, h);
}

}  // namespace

extern "C" {
int64_t fo_newton_schulz_workspace(const fo_matrix_shape* shapes, int64_t n_shapes) {
    if (int rc = validate_shapes(shapes, n_shapes)) return rc;
    int64_t most = 0;
    // lists of more shapes than a launch takes go through the workspace one part after the other
    for (int64_t i = 0; i < n_shapes; i += fo::kMaxShapes) {
        const int64_t n = n_shapes - i < fo::kMaxShapes ? n_shapes - i : fo::kMaxShapes;
        const int64_t bytes = plan(shapes + i, n, nullptr, nullptr);
        most = bytes > most ? bytes : most;
    }
    return most;
}

int fo_newton_schulz(const void* x, int dtype, int64_t count, int64_t rows, int64_t cols, int64_t stride, int64_t row_stride,
                     void* result, int steps, const float* coefficients, float eps, void* workspace, int64_t workspace_bytes,
                     void* stream) {
    if (dtype < FO_F32 || dtype > FO_F16) return fail(FO_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    if (count < 0 || rows < 0 || cols < 0 || count > INT32_MAX || rows > INT32_MAX || cols > INT32_MAX)
        return fail(FO_ERR_INVALID_ARGUMENT, "bad size");
    if (int rc = validate_iteration(steps, coefficients, eps)) return rc;
    const fo_matrix_shape shape{(int32_t)rows, (int32_t)cols, (int32_t)count, 0.0f};
    if (int rc = validate_shapes(&shape, 1)) return rc;
    if (count == 0 || rows == 0 || cols == 0) return 0;
    if (!x || !result || !workspace) return fail(FO_ERR_INVALID_ARGUMENT, "x, result and workspace must not be NULL");
    if ((uintptr_t)workspace & 255) return fail(FO_ERR_INVALID_ARGUMENT, "workspace must be aligned to 256 bytes");
    fo::Groups a{};
    if (workspace_bytes < plan(&shape, 1, (char*)workspace, &a)) return fail(FO_ERR_INVALID_ARGUMENT, "workspace too small");
    const fo::MatrixSource source{x, stride, row_stride};
    const Iteration it{steps, coefficients[0], coefficients[1], coefficients[2], eps};
    const fo::LastArgs last{(uint16_t*)result, nullptr, 0.0f};
    switch (dtype) {
        case FO_F32: return orthogonalise<fo::DT_F32>(a, source, it, last, (hipStream_t)stream);
        case FO_BF16: return orthogonalise<fo::DT_BF16>(a, source, it, last, (hipStream_t)stream);
        default: return orthogonalise<fo::DT_F16>(a, source, it, last, (hipStream_t)stream);
    }
}

int fo_muon_step(const fo_tensor_desc* matrices, const fo_matrix_shape* shapes, int64_t n_shapes, int dtype, int ecc_bytes,
                 int quantized, float keep, float momentum_coef, int nesterov, int steps, const float* coefficients, float eps,
                 void* workspace, int64_t workspace_bytes, void* stream) {
    if (dtype < FO_F32 || dtype > FO_F16) return fail(FO_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    if (ecc_bytes < 0 || ecc_bytes > 2) return fail(FO_ERR_INVALID_ARGUMENT, "ecc_bytes must be 0, 1 or 2, not %d", ecc_bytes);
    if (dtype == FO_F32 && ecc_bytes) return fail(FO_ERR_UNSUPPORTED, "fp32 parameters have no correction term");
    if (int rc = validate_iteration(steps, coefficients, eps)) return rc;
    if (int rc = validate_shapes(shapes, n_shapes)) return rc;
    const int64_t need = fo_newton_schulz_workspace(shapes, n_shapes);
    if (need == 0) return 0;
    if (!matrices || !workspace) return fail(FO_ERR_INVALID_ARGUMENT, "matrices and workspace must not be NULL");
    if ((uintptr_t)workspace & 255) return fail(FO_ERR_INVALID_ARGUMENT, "workspace must be aligned to 256 bytes");
    if (workspace_bytes < need) return fail(FO_ERR_INVALID_ARGUMENT, "workspace too small");
    const Iteration it{steps, coefficients[0], coefficients[1], coefficients[2], eps};
    for (int64_t i = 0; i < n_shapes; i += fo::kMaxShapes) {
        const int64_t n = n_shapes - i < fo::kMaxShapes ? n_shapes - i : fo::kMaxShapes;
        fo::Groups a{};
        plan(shapes + i, n, (char*)workspace, &a);
        if (a.n > 0) {
            const fo::MomentumArgs h{matrices, momentum_coef, 1.0f - momentum_coef, nesterov};
            const fo::LastArgs last{nullptr, matrices, keep};
            hipStream_t s = (hipStream_t)stream;
            if (int rc = dtype == FO_F32 ? momentum<fo::DT_F32>(a, h, quantized, s) : dtype == FO_BF16 ? momentum<fo::DT_BF16>(a, h, quantized, s)
                                                                                                : momentum<fo::DT_F16>(a, h, quantized, s)) return rc;
            if (int rc = launch_held_update(a, it, last, dtype, ecc_bytes, s)) return rc;
            if (a.n == 0) {
                for (int64_t k = 0; k < n; ++k) matrices += shapes[i + k].count;
                continue;
            }
            if (int rc = iterate<fo::DT_F32>(a, fo::MatrixSource{nullptr, 0, 0}, it, s, [&](fo::Groups& some, const fo::StepArgs& step, int cus) {
                    return launch_update(some, step, last, dtype, ecc_bytes, cus, s);
                })) return rc;
        }
        for (int64_t k = 0; k < n; ++k) matrices += shapes[i + k].count;
    }
    return 0;
}
}  // extern "C"
