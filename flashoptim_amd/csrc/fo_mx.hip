// Microscaled 4-bit floating point (MXFP4) for gfx950: quantiser, dequantiser and products, with their C entry points.
//
// Format.  A row is cut into groups of 32 values.  A group is stored as 32 E2M1 codes (sign, magnitudes 0, 0.5, 1, 1.5, 2, 3,
// 4, 6) and one E8M0 byte s, the power of two 2^(s - 127) that multiplies them.  With M the group's largest magnitude,
//     s - 127 = floor(log2 M) - 2, at least -127 (M = 0 included),     code = x / 2^(s - 127) rounded to nearest, ties to the even code,
// magnitudes above 6 (up to 8 occur) become 6.  A group that holds an infinity or a NaN has s = 255 and stands for NaNs, so that it
// shows in whatever is made of it.  Rows are filled up with zeros to whole blocks of 128 values: 64 bytes of codes, the first of two
// in the low half of a byte, and 4 scale bytes.
//
// A product contracts over rows of both operands, so the scales have to run along the contracted axis: the quantiser writes
// the row form of a matrix, the row form of its transpose, or both from one read.
#include "fo_gemm.h"
#include "fo_host.h"
#include "fo_mx.h"

namespace fo {

// Four pairs from memory, the first `valid` values of them, zeros after.
template <int DT> __device__ __forceinline__ void load_pairs(const char* p, int valid, Pair<DT> (&out)[4]) {
    constexpr int B = DTypeInfo<DT>::bytes, EPL = 16 / B;
    Pack<B, EPL> raw[B / 2];
#pragma unroll
    for (int i = 0; i < B / 2; ++i) load_piece<B, EPL>(raw[i], p + i * 16, valid - i * EPL);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (B == 2) out[i].v = raw[0].w[i];
        else { out[i].a = as_f32(raw[i / 2].w[i % 2 * 2]); out[i].b = as_f32(raw[i / 2].w[i % 2 * 2 + 1]); }
    }
}

struct QuantizeJob {
    const char* x;
    int64_t row_stride;   // in elements
    int rows, cols;
    uint8_t *codes, *scales;                  // of the rows, or null
    uint8_t *column_codes, *column_scales;    // of the columns, or null
};
struct QuantizeArgs {
    QuantizeJob job[2];
    int first_of_second;    // its first workgroup
};

// A 128 x 128 piece per workgroup: read once, all of it asked for before any of it is used; the row form out of registers (a
// group is four lanes), the column form through LDS (a thread takes 32 rows of a column, two neighbouring columns one after the
// other; four neighbouring threads write 64 adjacent bytes).  Bound by memory: 2 bytes in, 17/32 out per value and form; 14336 x 4096
// bf16 both ways in 47 us between other kernels (3.8 TB/s), in 39 after one of its kind on another matrix, one way in 29 to 33.
// The piece in LDS: rows an odd number of dwords apart, the lower half shifted so that the four groups of 32 rows that a wavefront reads
// at a time lie in different banks.
template <int B> struct QuantizePlaces {
    static constexpr int kStride = kBlock * B / 4 + 1, kShift = B == 2 ? 16 : 1, kDwords = kBlock * kStride + kShift;
    __device__ __forceinline__ static int of(int row) { return row * kStride + (row >> 6) * kShift; }
};
template <int DT, bool ROWS, bool COLUMNS> __global__ __launch_bounds__(256) void mx_quantize_kernel(QuantizeArgs args) {
    const bool second = (int)blockIdx.x >= args.first_of_second;
    const QuantizeJob& a = args.job[second];
    const int tile = (int)blockIdx.x - (second ? args.first_of_second : 0);
    constexpr int B = DTypeInfo<DT>::bytes;
    typedef QuantizePlaces<B> Places;
    extern __shared__ u32 lds[];
    const int tile_cols = (a.cols + kBlock - 1) / kBlock;
    const int row0 = tile / tile_cols * kBlock, col0 = tile % tile_cols * kBlock;
    const int64_t row_bytes = (int64_t)tile_cols * (kBlock / 2);
    const int piece = threadIdx.x & 15, line = threadIdx.x >> 4;
    const int col = col0 + piece * 8;
    Pair<DT> p[8][4];
    const char* x = a.x + (a.row_stride * (row0 + line) + col) * B;
    if (row0 + kBlock <= a.rows && col0 + kBlock <= a.cols) {
#pragma unroll
        for (int k = 0; k < 8; ++k) load_pairs<DT>(x + a.row_stride * k * 16 * B, 8, p[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) load_pairs<DT>(x + a.row_stride * k * 16 * B, row0 + line + k * 16 < a.rows ? a.cols - col : 0, p[k]);
    }
    if constexpr (COLUMNS) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            u32* out = lds + Places::of(k * 16 + line) + piece * 2 * B;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (B == 2) out[i] = p[k][i].v; else { out[2 * i] = as_u32(p[k][i].a); out[2 * i + 1] = as_u32(p[k][i].b); }
            }
        }
    }
    if (ROWS && a.codes) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int row = row0 + line + k * 16;
            u32 m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) { const u32 e = p[k][i].magnitude(); m = m > e ? m : e; }
            const u32 byte = scale_byte(largest_of_quad(m));
            const u32 w = byte == 255u ? 0u : encode8<DT>(p[k], scale_value(byte));
            if (row < a.rows) {
                *reinterpret_cast<u32*>(a.codes + row * row_bytes + col0 / 2 + piece * 4) = w;
                if ((piece & 3) == 0) a.scales[row * (row_bytes / 16) + col0 / kMxGroup + piece / 4] = (uint8_t)byte;
            }
        }
    }
    if constexpr (COLUMNS) {
        if (!a.column_codes) return;
        __syncthreads();
        const int64_t column_bytes = (int64_t)((a.rows + kBlock - 1) / kBlock) * (kBlock / 2);
        const int group = threadIdx.x & 3, pair = threadIdx.x >> 2;
        const u32* in = lds + Places::of(group * 32) + pair * (B / 2);
        u32 raw[32];   // both columns of a 16-bit type, the first of fp32
#pragma unroll
        for (int i = 0; i < 32; ++i) raw[i] = in[i * Places::kStride];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            Pair<DT> q[16];
            u32 m = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const u32 x = raw[2 * i], y = raw[2 * i + 1];
                if constexpr (B == 2) q[i].v = half ? __builtin_amdgcn_perm(y, x, 0x07060302u) : __builtin_amdgcn_perm(y, x, 0x05040100u);
                else { q[i].a = as_f32(x); q[i].b = as_f32(y); }
                const u32 e = q[i].magnitude();
                m = m > e ? m : e;
            }
            if constexpr (B == 4) {
                if (half == 0) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) raw[i] = in[i * Places::kStride + 1];
                }
            }
            const u32 byte = scale_byte(m);
            u32x4 w = {0, 0, 0, 0};
            if (byte != 255u) {
                const float scale = scale_value(byte);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = encode8<DT>(q + 4 * i, scale);
            }
            const int c = col0 + pair * 2 + half;
            if (c < a.cols) {
                *reinterpret_cast<u32x4*>(a.column_codes + c * column_bytes + row0 / 2 + group * 16) = w;
                a.column_scales[c * (column_bytes / 16) + row0 / kMxGroup + group] = (uint8_t)byte;
            }
        }
    }
}

// Eight values per thread.  Bound by memory: 14336 x 4096 to bf16 in 23 us, 6.5 TB/s.
template <int DT> __global__ __launch_bounds__(256) void mx_dequantize_kernel(const uint8_t* codes, const uint8_t* scales, char* out, int rows, int cols) {
    const int blocks = (cols + kBlock - 1) / kBlock, pieces = (cols + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = i / pieces;
    const int piece = (int)(i - row * pieces);
    if (row >= rows) return;
    const u32 w = *reinterpret_cast<const u32*>(codes + row * blocks * (kBlock / 2) + piece * 4);
    const u32 byte = scales[row * blocks * 4 + piece / 4];
    // the codes' values, then one product with the power of two, exact down to fp32's smallest numbers
    const float scale = byte == 255u ? __builtin_nanf("") : byte ? as_f32(byte << 23) : as_f32(0x00400000u);
    float v[8];
    const f32x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1);
    const f32x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
    v[0] = v0.x * scale; v[1] = v0.y * scale; v[2] = v1.x * scale; v[3] = v1.y * scale;
    v[4] = v2.x * scale; v[5] = v2.y * scale; v[6] = v3.x * scale; v[7] = v3.y * scale;
    store_values<DT>(v, out + (row * cols + piece * 8) * DTypeInfo<DT>::bytes, cols - piece * 8);
}

// ------------------------------------------------------------------------------------------------
// products
// ------------------------------------------------------------------------------------------------
struct ProductJob {
    const char *a, *b;                  // codes
    const uint8_t *a_scales, *b_scales;
    char* out;
    int rows, cols, blocks;             // of the result; 128-value blocks of the contracted axis
    int dtype;
    int64_t out_stride;                 // values between the result's rows
};
struct ProductArgs {
    ProductJob job[2];
    int seats_of_first;                 // of each die (fo_gemm.h)
};

struct ProductOut {
    static constexpr bool kColumns = false;
    char* out;
    int rows, cols, dtype;
    int64_t stride;
    struct In {};
    __device__ __forceinline__ void begin(int) const {}
    __device__ __forceinline__ void load(int, int, In&) const {}
    __device__ __forceinline__ void row(int i, int j, In, float (&v)[8]) const {
        if (i >= rows || j >= cols) return;
        const int64_t at = i * stride + j;
        if (dtype == DT_BF16) store_values<DT_BF16>(v, out + at * 2, cols - j);
        else if (dtype == DT_F16) store_values<DT_F16>(v, out + at * 2, cols - j);
        else store_values<DT_F32>(v, out + at * 4, cols - j);
    }
};

// Bound by the matrix cores: 4096 x 4096 over 32768 values in 231 us at least, 272 one after the other (4050 TFLOP/s); over 4096 values a round of 256 x 256 tiles takes 40 us,
// a quarter of it the start and the writing of the result.
template <int WT, int STAGES> __global__ __launch_bounds__(256, WT >= 96 ? 1 : 2) void mx_product_kernel(ProductArgs args) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef GemmTile<Mx4Product, WT, STAGES> Tile;
    const int seat = (int)(blockIdx.x >> 3);
    const bool second = seat >= args.seats_of_first;
    const ProductJob& p = args.job[second];
    const int rows = (p.rows + Tile::kTile - 1) / Tile::kTile, cols = (p.cols + Tile::kTile - 1) / Tile::kTile;
    const int64_t t = tile_of_seat(blockIdx.x & 7, seat - (second ? args.seats_of_first : 0), (int64_t)rows * cols);
    if (t < 0) return;
    int i, j;
    tile_at((int)t, rows, cols, i, j);
    const int64_t row_bytes = (int64_t)p.blocks * (kBlock / 2);
    const Operand a{p.a, row_bytes, p.a_scales, row_bytes / 16, p.rows}, b{p.b, row_bytes, p.b_scales, row_bytes / 16, p.cols};
    Tile tile(smem);
    tile.multiply(a, b, i * Tile::kTile, j * Tile::kTile, (int)row_bytes);
    ProductOut out{p.out, p.rows, p.cols, p.dtype, p.out_stride};
    tile.finish(i * Tile::kTile, j * Tile::kTile, out);
}

// Few rows against many: `tokens` <= 16 TILES rows of x, a weight of `cols` rows.  Bound by the weight's bytes, so what counts is
// how many of them are under way: a workgroup takes 16 ROWS weight rows, each of its eight wavefronts a run of blocks along the
// contracted axis, and asks for BATCH blocks (1 KiB of codes for 16 rows) before it looks at x.  The codes go straight from memory
// into the operand registers of 16x16x128 instructions (weight rows as their rows, tokens as their columns); the wavefronts add up
// through LDS at the end.  x comes as codes; or, with RAW, as values of type DT, which the workgroup quantises into LDS first, a
// group per thread: free beside the weight as long as it is a pass or two (kRawBlocks).  One token by 4096 x 14336 takes 11.5 us in all, 2.7
// TB/s of the weight; 16 tokens by 14336 x 4096 17.8 with their own quantiser's launch.
struct TokensArgs {
    const char* x;                 // codes, or values
    const uint8_t* x_scales;
    const char* weight;
    const uint8_t* weight_scales;
    char* out;
    int tokens, cols, inner, blocks;
    int64_t x_stride;              // RAW: elements between rows
    int dtype;                     // of the result
};
constexpr int kTokenWaves = 8, kTokenThreads = 64 * kTokenWaves;
constexpr int kRawBlocks = 256;    // most blocks of x that are quantised within the product: two groups per thread

template <int DT> __device__ __forceinline__ void quantise_tokens(const TokensArgs& p, char* codes, uint8_t* scales) {
    constexpr int B = DTypeInfo<DT>::bytes;
    for (int i = threadIdx.x; i < p.tokens * p.blocks * 4; i += kTokenThreads) {
        const int token = i / (p.blocks * 4), group = i - token * p.blocks * 4, at = group * kMxGroup;
        const char* x = p.x + (p.x_stride * token + at) * B;
        Pair<DT> q[4][4];
        u32 m = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) load_pairs<DT>(x + k * 8 * B, p.inner - at - k * 8, q[k]);
#pragma unroll
        for (int k = 0; k < 16; ++k) { const u32 e = q[k / 4][k % 4].magnitude(); m = m > e ? m : e; }
        const u32 byte = scale_byte(m);
        i32x4 v = {0, 0, 0, 0};
        if (byte != 255u) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = (int)encode8<DT>(q[k], scale_value(byte));
        }
        *reinterpret_cast<i32x4*>(codes + i * 16) = v;
        scales[i] = (uint8_t)byte;
    }
}

template <int DT, bool RAW, int TILES, int ROWS, int BATCH> __global__ __launch_bounds__(kTokenThreads) void mx_tokens_kernel(TokensArgs p) {
    constexpr int kAtOnce = TILES == 4 ? 2 : 4;   // blocks of x under way
    __shared__ f32x4 sums[kTokenWaves][ROWS * TILES][64];
    __shared__ __attribute__((aligned(16))) char raw_codes[RAW ? kRawBlocks * 64 : 16];
    __shared__ uint8_t raw_scales[RAW ? kRawBlocks * 4 : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int line = lane & 15, group = lane >> 4;
    // rows past the last, of the weight and of x, are read as copies of it: they make results that are not stored
    const char* w[ROWS];
    const uint8_t* ws[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        const int64_t want = ((int64_t)blockIdx.x * ROWS + r) * 16 + line, row = want < p.cols ? want : p.cols - 1;
        w[r] = p.weight + row * p.blocks * 64 + group * 16;
        ws[r] = p.weight_scales + row * p.blocks * 4 + group;
    }
    const char* x[TILES];
    const uint8_t* xs[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int token = t * 16 + line < p.tokens ? t * 16 + line : p.tokens - 1;
        x[t] = (RAW ? raw_codes : p.x) + (int64_t)token * p.blocks * 64 + group * 16;
        xs[t] = (RAW ? raw_scales : p.x_scales) + (int64_t)token * p.blocks * 4 + group;
    }
    const int per = (p.blocks + kTokenWaves - 1) / kTokenWaves;
    const int end = (wave + 1) * per < p.blocks ? (wave + 1) * per : p.blocks;
    f32x4 acc[ROWS][TILES];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int t = 0; t < TILES; ++t) acc[r][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    bool ready = !RAW;
    for (int first = wave * per; first < end || !ready; first += BATCH) {
        i32x4 wv[BATCH][ROWS];
        int wscale[BATCH][ROWS];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
            if (first + u < end) {
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    wv[u][r] = *reinterpret_cast<const i32x4*>(w[r] + (first + u) * 64);
                    wscale[u][r] = ws[r][(first + u) * 4];
                }
            }
        }
        if constexpr (RAW) {
            if (!ready) {   // every wavefront comes here once, in its first turn
                quantise_tokens<DT>(p, raw_codes, raw_scales);
                __syncthreads();
                ready = true;
            }
        }
#pragma unroll
        for (int part = 0; part < BATCH; part += kAtOnce) {
            i32x4 xv[kAtOnce][TILES];
            int xscale[kAtOnce][TILES];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (first + part + u < end) {
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        xv[u][t] = *reinterpret_cast<const i32x4*>(x[t] + (first + part + u) * 64);
                        xscale[u][t] = xs[t][(first + part + u) * 4];
                    }
                }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (first + part + u < end) {
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        const i32x8 vb = {xv[u][t].x, xv[u][t].y, xv[u][t].z, xv[u][t].w, 0, 0, 0, 0};
#pragma unroll
                        for (int r = 0; r < ROWS; ++r) {
                            const i32x4 c = wv[part + u][r];
                            const i32x8 va = {c.x, c.y, c.z, c.w, 0, 0, 0, 0};
                            acc[r][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, acc[r][t], 4, 4, 0, wscale[part + u][r], 0, xscale[u][t]);
                        }
                    }
                }
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int t = 0; t < TILES; ++t) sums[wave][r * TILES + t][lane] = acc[r][t];
    __syncthreads();
    for (int k = threadIdx.x; k < ROWS * TILES * 64; k += kTokenThreads) {
        const int piece = k >> 6, from = k & 63;
        f32x4 v = sums[0][piece][from];
#pragma unroll
        for (int s = 1; s < kTokenWaves; ++s) v += sums[s][piece][from];
        const int token = piece % TILES * 16 + (from & 15);
        const int64_t col = ((int64_t)blockIdx.x * ROWS + piece / TILES) * 16 + (from >> 4) * 4;
        if (token >= p.tokens) continue;
        const int64_t at = (int64_t)token * p.cols + col;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (col + e >= p.cols) break;
            if (p.dtype == DT_BF16) reinterpret_cast<__bf16*>(p.out)[at + e] = (__bf16)v[e];
            else if (p.dtype == DT_F16) reinterpret_cast<_Float16*>(p.out)[at + e] = (_Float16)v[e];
            else reinterpret_cast<float*>(p.out)[at + e] = v[e];
        }
    }
}

}  // namespace fo

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
namespace {
using namespace fo_host;

constexpr int64_t kMostWorkgroups = 1 << 22;
constexpr int64_t kMostLines = INT32_MAX - 255;
static_assert(FO_MXFP4_MOST_TOKENS == 64, "four tiles of 16");

int validate_matrix(const char* what, int64_t rows, int64_t cols, int dtype) {
    if (rows < 0 || cols < 0) return fail(FO_ERR_INVALID_ARGUMENT, "%s: negative size", what);
    if (rows > kMostLines || cols > kMostLines) return fail(FO_ERR_UNSUPPORTED, "%s: %lld x %lld is too large", what, (long long)rows, (long long)cols);
    if (dtype < FO_F32 || dtype > FO_F16) return fail(FO_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    return 0;
}

// What the lanes' 32-bit offsets into a tile's rows reach.
int validate_inner(const char* what, int64_t inner) {
    if (inner == 0) return fail(FO_ERR_UNSUPPORTED, "%s: nothing to contract over", what);
    if (inner > 1 << 24) return fail(FO_ERR_UNSUPPORTED, "%s: rows of %lld values are too long", what, (long long)inner);
    return 0;
}

int64_t blocks_of(int64_t n) { return (n + fo::kBlock - 1) / fo::kBlock; }

template <class K, class... Args> int launch(K kernel, int64_t grid, int threads, int lds, void* stream, const char* what, Args... args) {
    if (grid > kMostWorkgroups) return fail(FO_ERR_UNSUPPORTED, "%s: %lld workgroups are more than one launch takes", what, (long long)grid);
    if (lds > 65536) {
        if (int rc = check_hip(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, lds), what)) return rc;
    }
    kernel<<<dim3((unsigned)grid), dim3(threads), lds, (hipStream_t)stream>>>(args...);
    return check_hip(hipGetLastError(), what);
}

// One matrix and where its forms go: codes, then scales.
fo::QuantizeJob quantize_job(const void* x, int64_t rows, int64_t cols, int64_t row_stride, void* codes, void* scales, void* column_codes, void* column_scales) {
    return {(const char*)x, row_stride, (int)rows, (int)cols, (uint8_t*)codes, (uint8_t*)scales, (uint8_t*)column_codes, (uint8_t*)column_scales};
}
int64_t form_codes(int64_t rows, int64_t cols) { return rows * blocks_of(cols) * 64; }
int64_t form_bytes(int64_t rows, int64_t cols) { return (rows * blocks_of(cols) * 68 + 255) / 256 * 256; }

template <int DT> int launch_quantize(const fo::QuantizeJob* jobs, int n, void* stream) {
    constexpr int kLds = fo::QuantizePlaces<fo::DTypeInfo<DT>::bytes>::kDwords * 4;
    const char* what = "fo_mxfp4_quantize";
    fo::QuantizeArgs a{};
    int64_t grid = 0;
    bool rows = false, columns = false;
    for (int i = 0; i < n; ++i) {
        a.job[i] = jobs[i];
        if (i == 1) a.first_of_second = (int)grid;
        grid += blocks_of(jobs[i].rows) * blocks_of(jobs[i].cols);
        if (grid > kMostWorkgroups) return fail(FO_ERR_UNSUPPORTED, "%s: too many values for one launch", what);
        rows |= jobs[i].codes != nullptr;
        columns |= jobs[i].column_codes != nullptr;
    }
    if (n == 1) a.first_of_second = (int)grid;
    if (!columns) return launch(fo::mx_quantize_kernel<DT, true, false>, grid, 256, 0, stream, what, a);
    if (!rows) return launch(fo::mx_quantize_kernel<DT, false, true>, grid, 256, kLds, stream, what, a);
    return launch(fo::mx_quantize_kernel<DT, true, true>, grid, 256, kLds, stream, what, a);
}
int launch_quantize(int dtype, const fo::QuantizeJob* jobs, int n, void* stream) {
    if (dtype == FO_F32) return launch_quantize<fo::DT_F32>(jobs, n, stream);
    return dtype == FO_BF16 ? launch_quantize<fo::DT_BF16>(jobs, n, stream) : launch_quantize<fo::DT_F16>(jobs, n, stream);
}

template <int DT, bool RAW, int TILES, int ROWS> int launch_tokens(const fo::TokensArgs& p, void* stream) {
    const int64_t grid = (p.cols + 16 * ROWS - 1) / (16 * ROWS);
    const char* what = RAW ? "fo_mxfp4_tokens" : "fo_mxfp4_product";
    // a wavefront's run in one batch where it fits
    if (p.blocks <= 4 * fo::kTokenWaves) return launch(fo::mx_tokens_kernel<DT, RAW, TILES, ROWS, 4>, grid, fo::kTokenThreads, 0, stream, what, p);
    return launch(fo::mx_tokens_kernel<DT, RAW, TILES, ROWS, 16 / ROWS>, grid, fo::kTokenThreads, 0, stream, what, p);
}
// Two pieces of 16 weight rows to a workgroup read x half as often, where that leaves every compute unit a workgroup: 13.2 us
// for 16 tokens by 14336 x 4096 against 16.1, 26.2 against 37.6 for 64; with 4096 rows (half the compute units) 38.8 against 32.8.
bool by_two(const fo::TokensArgs& p) { return p.cols >= 32 * compute_units(); }

template <int DT> int launch_raw_tokens(const fo::TokensArgs& p, void* stream) {
    if (p.tokens <= 16) return by_two(p) ? launch_tokens<DT, true, 1, 2>(p, stream) : launch_tokens<DT, true, 1, 1>(p, stream);
    return p.tokens <= 32 ? launch_tokens<DT, true, 2, 1>(p, stream) : launch_tokens<DT, true, 4, 1>(p, stream);
}
template <int TILES> int launch_coded_tokens(const fo::TokensArgs& p, void* stream) {
    return by_two(p) ? launch_tokens<fo::DT_BF16, false, TILES, 2>(p, stream) : launch_tokens<fo::DT_BF16, false, TILES, 1>(p, stream);
}
int launch_coded_tokens(const fo::TokensArgs& p, void* stream) {
    if (p.tokens <= 16) return launch_coded_tokens<1>(p, stream);
    return p.tokens <= 32 ? launch_coded_tokens<2>(p, stream) : launch_coded_tokens<4>(p, stream);
}

// Times of 4096 x 4096 products (3840 x 3840 for 192 x 192 tiles) over 1024 to 16384 values: a 256 x 256 tile takes 40 us over 4096 and
// 130 over 16384, two 128 x 128 tiles on a compute unit 26 and 90 (alone 18 and 62), five 64 x 64 21 and 75 (two of them 13 and 44).
constexpr fo::TileCost kTileCosts[] = {
    {128, 2, 1, 11.5, 0.0073, 11.5, 0.0073}, {96, 3, 1, 8.0, 0.0046, 8.0, 0.0046}, {64, 2, 2, 3.5, 0.0036, 5.0, 0.0052},
    {32, 2, 5, 2.0, 0.0022, 5.0, 0.0043}, {32, 4, 2, 2.0, 0.0012, 2.2, 0.0024}};

int64_t tiles(const fo::ProductJob& p, int wt) { return fo::tiles_of(p.rows, p.cols, wt); }

template <int WT, int STAGES> int launch_products(const fo::ProductJob* jobs, int n, void* stream) {
    fo::ProductArgs a{};
    int64_t seats = 0;
    for (int i = 0; i < n; ++i) {
        a.job[i] = jobs[i];
        if (i == 1) a.seats_of_first = (int)seats;
        seats += fo::seats_of(tiles(jobs[i], WT));
        if (seats > kMostWorkgroups) return fail(FO_ERR_UNSUPPORTED, "fo_mxfp4_product: too large a result for one launch");
    }
    if (n == 1) a.seats_of_first = (int)seats;
    return launch(fo::mx_product_kernel<WT, STAGES>, 8 * seats, 256, fo::GemmTile<fo::Mx4Product, WT, STAGES>::kLds, stream, "fo_mxfp4_product", a);
}

int launch_products(const fo::TileCost& t, const fo::ProductJob* jobs, int n, void* stream) {
    switch (t.wt) {
        case 128: return launch_products<128, 2>(jobs, n, stream);
        case 96: return launch_products<96, 3>(jobs, n, stream);
        case 64: return launch_products<64, 2>(jobs, n, stream);
        default: return t.stages == 4 ? launch_products<32, 4>(jobs, n, stream) : launch_products<32, 2>(jobs, n, stream);
    }
}
// The first `at` rows (columns) of a product, and the others.  Codes of rows are multiples of 64 bytes, so all stays aligned.
void divide(const fo::ProductJob& p, bool columns, int at, fo::ProductJob& first, fo::ProductJob& rest) {
    const int64_t row_bytes = (int64_t)p.blocks * (fo::kBlock / 2);
    first = rest = p;
    (columns ? first.cols : first.rows) = at;
    (columns ? rest.cols : rest.rows) -= at;
    (columns ? rest.b : rest.a) += at * row_bytes;
    (columns ? rest.b_scales : rest.a_scales) += at * (row_bytes / 16);
    rest.out += (columns ? (int64_t)at : (int64_t)at * p.out_stride) * (p.dtype == fo::DT_F32 ? 4 : 2);
}

// Up to two products in one launch, the longer contraction first; the last one may be cut (fo_gemm.h).
int launch_products(fo::ProductJob* jobs, int n, void* stream) {
    const int cus = compute_units();
    if (cus <= 0) return fail(FO_ERR_NO_DEVICE, "no device");
    if (n == 2 && jobs[0].blocks < jobs[1].blocks) { const fo::ProductJob t = jobs[0]; jobs[0] = jobs[1]; jobs[1] = t; }
    const fo::ProductJob last = jobs[n - 1];
    const fo::Cut cut = fo::best_cut(kTileCosts, last.rows, last.cols, (double)last.blocks * fo::kBlock,
                                     [&](int wt) { return n == 2 ? (double)tiles(jobs[0], wt) : 0.0; }, (double)jobs[0].blocks * fo::kBlock, cus);
    if (!cut.rest.wt) return launch_products(cut.tile, jobs, n, stream);
    fo::ProductJob rest;
    divide(last, cut.columns, cut.lines * 2 * cut.tile.wt, jobs[n - 1], rest);
    if (int rc = launch_products(cut.tile, jobs, n, stream)) return rc;
    return launch_products(cut.rest, &rest, 1, stream);
}

fo::TokensArgs tokens_of(const fo::ProductJob& p) {
    return {p.a, p.a_scales, p.b, p.b_scales, p.out, p.rows, p.cols, p.blocks * fo::kBlock, p.blocks, 0, p.dtype};
}
// The kernel for few rows for those that have few, one launch for the others.
int run_products(const fo::ProductJob* jobs, int n, void* stream) {
    fo::ProductJob large[2];
    int k = 0;
    for (int i = 0; i < n; ++i) {
        if (jobs[i].rows > FO_MXFP4_MOST_TOKENS) { large[k++] = jobs[i]; continue; }
        if (int rc = launch_coded_tokens(tokens_of(jobs[i]), stream)) return rc;
    }
    return k ? launch_products(large, k, stream) : 0;
}

// A product of two forms: codes, then scales.
fo::ProductJob product_of(const void* a, int64_t rows, const void* b, int64_t cols, int64_t inner, void* out, int dtype) {
    return {(const char*)a, (const char*)b, (const uint8_t*)a + form_codes(rows, inner), (const uint8_t*)b + form_codes(cols, inner), (char*)out,
            (int)rows, (int)cols, (int)blocks_of(inner), dtype, cols};
}

int check_forms(const void* a, const void* b, const void* c) {
    if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) return fail(FO_ERR_INVALID_ARGUMENT, "forms and workspace must be aligned to 16 bytes");
    return 0;
}

}  // namespace

extern "C" {
int fo_mxfp4_quantize(const void* x, int dtype, int64_t rows, int64_t cols, int64_t row_stride, void* codes, void* scales,
                      void* column_codes, void* column_scales, void* stream) {
    if (int rc = validate_matrix("fo_mxfp4_quantize", rows, cols, dtype)) return rc;
    if (!codes != !scales || !column_codes != !column_scales || (!codes && !column_codes))
        return fail(FO_ERR_INVALID_ARGUMENT, "codes and scales of the rows, of the columns or of both must be given");
    if (rows == 0 || cols == 0) return 0;
    if (!x) return fail(FO_ERR_INVALID_ARGUMENT, "x must not be NULL");
    if (((uintptr_t)codes | (uintptr_t)column_codes) & 15) return fail(FO_ERR_INVALID_ARGUMENT, "codes must be aligned to 16 bytes");
    const fo::QuantizeJob job = quantize_job(x, rows, cols, row_stride, codes, scales, column_codes, column_scales);
    return launch_quantize(dtype, &job, 1, stream);
}

int fo_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t cols, void* out, int dtype, void* stream) {
    if (int rc = validate_matrix("fo_mxfp4_dequantize", rows, cols, dtype)) return rc;
    if (rows == 0 || cols == 0) return 0;
    if (!codes || !scales || !out) return fail(FO_ERR_INVALID_ARGUMENT, "codes, scales and out must not be NULL");
    if ((uintptr_t)codes & 3) return fail(FO_ERR_INVALID_ARGUMENT, "codes must be aligned to 4 bytes");
    const int64_t grid = (rows * ((cols + 7) / 8) + 255) / 256;
    const char* what = "fo_mxfp4_dequantize";
    switch (dtype) {
        case FO_F32: return launch(fo::mx_dequantize_kernel<fo::DT_F32>, grid, 256, 0, stream, what, (const uint8_t*)codes, (const uint8_t*)scales, (char*)out, (int)rows, (int)cols);
        case FO_BF16: return launch(fo::mx_dequantize_kernel<fo::DT_BF16>, grid, 256, 0, stream, what, (const uint8_t*)codes, (const uint8_t*)scales, (char*)out, (int)rows, (int)cols);
        default: return launch(fo::mx_dequantize_kernel<fo::DT_F16>, grid, 256, 0, stream, what, (const uint8_t*)codes, (const uint8_t*)scales, (char*)out, (int)rows, (int)cols);
    }
}

int fo_mxfp4_product(const void* a, const void* a_scales, int64_t rows, const void* b, const void* b_scales, int64_t cols, int64_t inner,
                     void* out, int dtype, void* stream) {
    if (int rc = validate_matrix("fo_mxfp4_product", rows, cols, dtype)) return rc;
    if (int rc = validate_matrix("fo_mxfp4_product", rows, inner, dtype)) return rc;
    if (rows == 0 || cols == 0) return 0;
    if (int rc = validate_inner("fo_mxfp4_product", inner)) return rc;
    if (!a || !a_scales || !b || !b_scales || !out) return fail(FO_ERR_INVALID_ARGUMENT, "operands and out must not be NULL");
    if (((uintptr_t)a | (uintptr_t)b) & 15 || ((uintptr_t)a_scales | (uintptr_t)b_scales) & 3)
        return fail(FO_ERR_INVALID_ARGUMENT, "codes must be aligned to 16 bytes, scales to 4");
    const fo::ProductJob job{(const char*)a, (const char*)b, (const uint8_t*)a_scales, (const uint8_t*)b_scales, (char*)out, (int)rows, (int)cols, (int)blocks_of(inner), dtype, cols};
    return run_products(&job, 1, stream);
}

int64_t fo_mxfp4_tokens_workspace(int64_t tokens, int64_t inner) {
    if (int rc = validate_matrix("fo_mxfp4_tokens", tokens, inner, FO_F32)) return rc;
    const int64_t blocks = tokens * blocks_of(inner);
    return blocks <= fo::kRawBlocks ? 0 : blocks * 68;
}

int fo_mxfp4_tokens(const void* x, int x_dtype, int64_t tokens, int64_t row_stride, const void* weight, const void* weight_scales, int64_t cols,
                    int64_t inner, void* out, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
    if (int rc = validate_matrix("fo_mxfp4_tokens", tokens, cols, dtype)) return rc;
    if (int rc = validate_matrix("fo_mxfp4_tokens", tokens, inner, x_dtype)) return rc;
    if (tokens > FO_MXFP4_MOST_TOKENS) return fail(FO_ERR_UNSUPPORTED, "fo_mxfp4_tokens takes at most %d rows, not %lld", FO_MXFP4_MOST_TOKENS, (long long)tokens);
    if (tokens == 0 || cols == 0) return 0;
    if (int rc = validate_inner("fo_mxfp4_tokens", inner)) return rc;
    if (!x || !weight || !weight_scales || !out) return fail(FO_ERR_INVALID_ARGUMENT, "operands and out must not be NULL");
    if ((uintptr_t)weight & 15) return fail(FO_ERR_INVALID_ARGUMENT, "codes must be aligned to 16 bytes");
    const int64_t need = fo_mxfp4_tokens_workspace(tokens, inner), blocks = blocks_of(inner);
    fo::TokensArgs p{(const char*)x, nullptr, (const char*)weight, (const uint8_t*)weight_scales, (char*)out, (int)tokens, (int)cols, (int)inner, (int)blocks, row_stride, dtype};
    if (need > 0) {
        if (!workspace || workspace_bytes < need || (uintptr_t)workspace & 15)
            return fail(FO_ERR_INVALID_ARGUMENT, "a workspace of %lld bytes, aligned to 16, is needed", (long long)need);
        p.x = (const char*)workspace;
        p.x_scales = (const uint8_t*)workspace + tokens * blocks * 64;
        if (int rc = fo_mxfp4_quantize(x, x_dtype, tokens, inner, row_stride, workspace, (uint8_t*)workspace + tokens * blocks * 64, nullptr, nullptr, stream)) return rc;
        return launch_coded_tokens(p, stream);
    }
    switch (x_dtype) {
        case FO_F32: return launch_raw_tokens<fo::DT_F32>(p, stream);
        case FO_BF16: return launch_raw_tokens<fo::DT_BF16>(p, stream);
        default: return launch_raw_tokens<fo::DT_F16>(p, stream);
    }
}

int64_t fo_mxfp4_form_bytes(int64_t rows, int64_t cols) {
    if (int rc = validate_matrix("fo_mxfp4_form_bytes", rows, cols, FO_F32)) return rc;
    return form_bytes(rows, cols);
}

int fo_mxfp4_linear_forward(const void* x, int x_dtype, int64_t tokens, int64_t x_stride, const void* weight, int weight_dtype, int64_t outer,
                            int64_t weight_stride, int64_t inner, void* x_columns, void* weight_columns, void* out, void* workspace,
                            int64_t workspace_bytes, void* stream) {
    const char* what = "fo_mxfp4_linear_forward";
    if (int rc = validate_matrix(what, tokens, inner, x_dtype)) return rc;
    if (int rc = validate_matrix(what, outer, inner, weight_dtype)) return rc;
    if (tokens == 0 || outer == 0) return fail(FO_ERR_UNSUPPORTED, "%s: an empty product", what);
    if (int rc = validate_inner(what, inner)) return rc;
    if (!x || !weight || !out || !workspace) return fail(FO_ERR_INVALID_ARGUMENT, "x, weight, out and workspace must not be NULL");
    if (int rc = check_forms(x_columns, weight_columns, workspace)) return rc;
    const int64_t x_form = form_bytes(tokens, inner);
    if (workspace_bytes < x_form + form_bytes(outer, inner)) return fail(FO_ERR_INVALID_ARGUMENT, "workspace too small");
    char *xr = (char*)workspace, *wr = xr + x_form;
    const fo::QuantizeJob jobs[2] = {
        quantize_job(x, tokens, inner, x_stride, xr, xr + form_codes(tokens, inner), x_columns, x_columns ? (char*)x_columns + form_codes(inner, tokens) : nullptr),
        quantize_job(weight, outer, inner, weight_stride, wr, wr + form_codes(outer, inner), weight_columns, weight_columns ? (char*)weight_columns + form_codes(inner, outer) : nullptr)};
    if (x_dtype == weight_dtype) {
        if (int rc = launch_quantize(x_dtype, jobs, 2, stream)) return rc;
    } else {
        if (int rc = launch_quantize(x_dtype, jobs, 1, stream)) return rc;
        if (int rc = launch_quantize(weight_dtype, jobs + 1, 1, stream)) return rc;
    }
    const fo::ProductJob y = product_of(xr, tokens, wr, outer, inner, out, x_dtype);
    return run_products(&y, 1, stream);
}

int fo_mxfp4_linear_backward(const void* dy, int dy_dtype, int64_t tokens, int64_t dy_stride, int64_t outer, int64_t inner, const void* x_columns,
                             const void* weight_columns, void* dx, int dx_dtype, void* dw, int dw_dtype, void* workspace, int64_t workspace_bytes,
                             void* stream) {
    const char* what = "fo_mxfp4_linear_backward";
    if (int rc = validate_matrix(what, tokens, outer, dy_dtype)) return rc;
    if (int rc = validate_matrix(what, outer, inner, dx_dtype)) return rc;
    if (int rc = validate_matrix(what, tokens, inner, dw_dtype)) return rc;
    if (tokens == 0 || inner == 0) return fail(FO_ERR_UNSUPPORTED, "%s: an empty product", what);
    if (int rc = validate_inner(what, outer)) return rc;
    if (int rc = validate_inner(what, tokens)) return rc;
    if (!dy || !workspace || !dx != !weight_columns || !dw != !x_columns || (!dx && !dw))
        return fail(FO_ERR_INVALID_ARGUMENT, "dy, workspace, and dx with weight_columns or dw with x_columns or both must be given");
    if (int rc = check_forms(x_columns, weight_columns, workspace)) return rc;
    const int64_t row_form = dx ? form_bytes(tokens, outer) : 0;
    if (workspace_bytes < row_form + (dw ? form_bytes(outer, tokens) : 0)) return fail(FO_ERR_INVALID_ARGUMENT, "workspace too small");
    char* rows = dx ? (char*)workspace : nullptr;
    char* columns = dw ? (char*)workspace + row_form : nullptr;
    const fo::QuantizeJob job = quantize_job(dy, tokens, outer, dy_stride, rows, rows ? rows + form_codes(tokens, outer) : nullptr, columns,
                                             columns ? columns + form_codes(outer, tokens) : nullptr);
    if (int rc = launch_quantize(dy_dtype, &job, 1, stream)) return rc;
    fo::ProductJob products[2];
    int n = 0;
    if (dx) products[n++] = product_of(rows, tokens, weight_columns, inner, outer, dx, dx_dtype);
    if (dw) products[n++] = product_of(columns, outer, x_columns, inner, tokens, dw, dw_dtype);
    return run_products(products, n, stream);
}
}  // extern "C"
