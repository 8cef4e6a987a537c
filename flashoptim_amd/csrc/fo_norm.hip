// Root-mean-square norm of a residual stream's rows, with the addition that makes them, its gradients, and its output in MXFP4.
//
//   s = x + r (rounded to r's type: the stream that goes on; without r, s = x)        n = s / sqrt(mean(s^2) + eps)       y = n w
//   dn = dy w      ds = (dn - n mean(dn n)) / sqrt(mean(s^2) + eps) + ds'              dx = dr = ds                        dw = sum over rows of dy n
//
// with ds' the gradient that the stream brings along.  The norm reads the stream as it is stored, so the backward pass finds the same
// numbers; everything else is held in fp32 and rounded once.  Kept for the backward pass: the stream and one fp32 number a row.
//
// A row is held in registers by one workgroup from its load to its store: every byte moves once.  Values that a wavefront holds go by
// eight neighbours to a lane whatever the type, so that the sums, and with them the results, do not go by the type's width.
#include "fo_gemm.h"
#include "fo_host.h"
#include "fo_mx.h"

namespace fo {

struct NormArgs {
    const char* x;
    const char* residual;     // null: none
    const char* weight;       // null: ones
    char* stream;             // x + residual, contiguous; null without a residual
    char* y;                  // contiguous rows, or MXFP4 codes
    uint8_t* scales;          // of MXFP4
    float* inverse;           // 1 / sqrt(mean(s^2) + eps) of each row, or null
    int64_t x_stride, residual_stride, rows;
    int cols, weight_dtype;
    float eps;
};
struct NormGradArgs {
    const char* s;            // the stream (x where there is no residual)
    const char* weight;
    const float* inverse;
    const char* dy;
    const char* dstream;      // null: none
    char *dx, *dresidual;     // contiguous; null: not wanted
    float* partial;           // a row of `cols` sums per workgroup, or null
    int64_t s_stride, dy_stride, dstream_stride, rows;
    int cols, weight_dtype;
};

__device__ __forceinline__ void load_any(float (&v)[8], const char* p, int dtype, int at, int valid) {
    if (dtype == DT_F32) load_values<DT_F32>(v, p + (int64_t)at * 4, valid);
    else if (dtype == DT_BF16) load_values<DT_BF16>(v, p + (int64_t)at * 2, valid);
    else load_values<DT_F16>(v, p + (int64_t)at * 2, valid);
}

// Stores eight values rounded to RT and leaves in `v` what was stored (one conversion for both: compilers may join the rounding of a
// sum to fp32 with a second one in one use of it and not in another).
template <int RT> __device__ __forceinline__ void store_rounded(float (&v)[8], char* p, int valid) {
    constexpr int B = DTypeInfo<RT>::bytes, EPL = 16 / B;
#pragma unroll
    for (int part = 0; part < 8 / EPL; ++part) {
        Pack<B, EPL> d;
#pragma unroll
        for (int k = 0; k < EPL; k += 2) {
            float a, b;
            narrow_pair<RT, EPL>(d, k, v[part * EPL + k], v[part * EPL + k + 1], a, b);
        }
        store_piece<B, EPL>(d, p + part * 16, valid - part * EPL);
#pragma unroll
        for (int k = 0; k < EPL; ++k) v[part * EPL + k] = widen<RT, EPL>(d, k);
    }
}

template <int CTRL> __device__ __forceinline__ float from_lane(float x) {
    return as_f32((u32)__builtin_amdgcn_mov_dpp((int)as_u32(x), CTRL, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ double from_lane(double x) {
    const u32x2 v = __builtin_bit_cast(u32x2, x);
    const u32x2 w = {(u32)__builtin_amdgcn_mov_dpp((int)v.x, CTRL, 0xf, 0xf, true), (u32)__builtin_amdgcn_mov_dpp((int)v.y, CTRL, 0xf, 0xf, true)};
    return __builtin_bit_cast(double, w);
}
__device__ __forceinline__ float read_lane(float x, int lane) { return as_f32((u32)__builtin_amdgcn_readlane((int)as_u32(x), lane)); }
__device__ __forceinline__ double read_lane(double x, int lane) {
    const u32x2 v = __builtin_bit_cast(u32x2, x);
    const u32x2 w = {(u32)__builtin_amdgcn_readlane((int)v.x, lane), (u32)__builtin_amdgcn_readlane((int)v.y, lane)};
    return __builtin_bit_cast(double, w);
}
// The sum over a wavefront, the same in every lane.
template <class T> __device__ __forceinline__ T wave_sum(T x) {
    x += from_lane<0xb1>(x);     // lanes 1 0 3 2
    x += from_lane<0x4e>(x);     // lanes 2 3 0 1
    x += from_lane<0x141>(x);    // eight lanes mirrored
    x += from_lane<0x140>(x);    // sixteen lanes mirrored
    return (read_lane(x, 0) + read_lane(x, 16)) + (read_lane(x, 32) + read_lane(x, 48));
}

// The sum over a workgroup, the same in every thread.  `places` takes turns between two arrays, so one barrier is enough.
template <int THREADS, class T> __device__ __forceinline__ T group_sum(T x, T (&places)[2][16], int& turn) {
    x = wave_sum(x);
    if constexpr (THREADS == 64) return x;
    T(&mine)[16] = places[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) mine[threadIdx.x >> 6] = x;
    __syncthreads();
    T all = mine[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) all += mine[w];
    return all;
}

// 1 / sqrt(mean(s^2) + eps).  Squares are added in fp64, which costs nothing beside the loads and holds the squares of every fp32 number, and rounded to fp32 as a
// mean; only where that is no normal number is the root taken in fp64 too.
template <int THREADS, int V> __device__ __forceinline__ float inverse_root(const float (&s)[V][8], int cols, float eps, double (&places)[2][16], int& turn) {
    double sum = 0.0;
#pragma unroll
    for (int p = 0; p < V; ++p)
#pragma unroll
        for (int k = 0; k < 8; ++k) sum = __builtin_fma((double)s[p][k], (double)s[p][k], sum);
    sum = group_sum<THREADS>(sum, places, turn) / cols;
    const float mean = (float)sum + eps;
    if (mean >= 0x1p-120f && mean <= 0x1p126f) return rsqrtf(mean);
    return (float)(1.0 / __builtin_sqrt(sum + (double)eps));
}

// What a thread holds of a row as it came from memory: V pieces of eight values.  WHOLE: rows are whole multiples of eight, so a piece is there or it is not.
template <int DT, int THREADS, int V, bool WHOLE> struct Raw {
    static constexpr int B = DTypeInfo<DT>::bytes, EPL = 16 / B;
    Pack<B, EPL> d[V][8 / EPL];
    __device__ __forceinline__ void load(const char* row, int cols) {
#pragma unroll
        for (int p = 0; p < V; ++p) {
            const int c = (threadIdx.x + p * THREADS) * 8;
#pragma unroll
            for (int part = 0; part < 8 / EPL; ++part) {
#pragma unroll
                for (int k = 0; k < Pack<B, EPL>::kDwords; ++k) d[p][part].w[k] = 0;
                if (c < cols) load_piece<B, EPL>(d[p][part], row + ((int64_t)c + part * EPL) * B, WHOLE ? EPL : cols - c - part * EPL);
            }
        }
    }
    __device__ __forceinline__ float value(int p, int k) const { return widen<DT, EPL>(d[p][k / EPL], k % EPL); }
};

// XT: type of x and y, RT: of the residual and the stream.  THREADS hold V pieces of eight values each, THREADS * V * 8 >= cols.  A workgroup takes every
// gridDim.x-th row and asks for the next one before it adds up the squares of this one (rows of up to 8192 values; longer ones leave no registers
// for that: 2048 x 16384 and 4096 x 8200 bf16 in 45 us, as 4096 x 8192, and back in 57 where 4096 x 8192 takes 51).
// Bound by memory: 8192 x 4096 bf16 with a residual in 42 us (6.4 TB/s; 56 without the next row ahead), into MXFP4 4096 of them in 18; one row 2.8 us, a launch.
template <int XT, int RT, int THREADS, int V, bool MX, bool WHOLE> __global__ __launch_bounds__(THREADS) void norm_kernel(NormArgs a) {
    constexpr int XB = DTypeInfo<XT>::bytes, RB = DTypeInfo<RT>::bytes;
    constexpr bool kAhead = THREADS <= 256;
    __shared__ double places[2][16];
    int turn = 0;
    const int cols = a.cols, first = threadIdx.x * 8;
    Raw<XT, THREADS, V, WHOLE> x;
    Raw<RT, THREADS, V, WHOLE> r;
    x.load(a.x + blockIdx.x * a.x_stride * XB, cols);
    if (a.residual) r.load(a.residual + blockIdx.x * a.residual_stride * RB, cols);
    float w[V][8];
#pragma unroll
    for (int p = 0; p < V; ++p) {
        const int c = first + p * THREADS * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k) w[p][k] = 1.0f;
        if (a.weight && c < cols) load_any(w[p], a.weight, a.weight_dtype, c, WHOLE ? 8 : cols - c);
    }
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        float s[V][8];
#pragma unroll
        for (int p = 0; p < V; ++p) {
            const int c = first + p * THREADS * 8;
#pragma unroll
            for (int k = 0; k < 8; ++k) s[p][k] = x.value(p, k);
            if (a.residual) {
#pragma unroll
                for (int k = 0; k < 8; ++k) s[p][k] += r.value(p, k);
                if (c < cols) store_rounded<RT>(s[p], a.stream + (row * cols + c) * RB, WHOLE ? 8 : cols - c);
            }
        }
        const int64_t next = row + gridDim.x;
        if (kAhead && next < a.rows) {
            x.load(a.x + next * a.x_stride * XB, cols);
            if (a.residual) r.load(a.residual + next * a.residual_stride * RB, cols);
        }
        const float inverse = inverse_root<THREADS, V>(s, cols, a.eps, places, turn);
        if (a.inverse && threadIdx.x == 0) a.inverse[row] = inverse;
#pragma unroll
        for (int p = 0; p < V; ++p) {
            const int c = first + p * THREADS * 8;
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] = s[p][k] * inverse * w[p][k];
            if constexpr (MX) {
                const int blocks = (cols + kBlock - 1) / kBlock;
                if (c >= blocks * kBlock) continue;    // quads stay together: blocks are sixteen lanes
                Pair<DT_F32> q[4];
                u32 m = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    q[k].a = c + 2 * k < cols ? y[2 * k] : 0.0f;
                    q[k].b = c + 2 * k + 1 < cols ? y[2 * k + 1] : 0.0f;
                    const u32 e = q[k].magnitude();
                    m = m > e ? m : e;
                }
                const u32 byte = scale_byte(largest_of_quad(m));
                const u32 codes = byte == 255u ? 0u : encode8<DT_F32>(q, scale_value(byte));
                *reinterpret_cast<u32*>(a.y + row * blocks * (kBlock / 2) + c / 2) = codes;
                if ((threadIdx.x & 3) == 0) a.scales[row * blocks * 4 + c / kMxGroup] = (uint8_t)byte;
            } else {
                if (c < cols) store_values<XT>(y, a.y + (row * cols + c) * XB, WHOLE ? 8 : cols - c);
            }
        }
        if (!kAhead && next < a.rows) {
            x.load(a.x + next * a.x_stride * XB, cols);
            if (a.residual) r.load(a.residual + next * a.residual_stride * RB, cols);
        }
    }
}

// The same way back; what a row adds to dw stays in registers until the end.  Bound by memory: 8192 x 4096 bf16 in 52 us (5.2 TB/s; 78 without the next row ahead), with two
// workgroups to a compute unit (one 70, four 62: their rows of partial sums have to be written and read).
template <int XT, int RT, int THREADS, int V, bool WHOLE> __global__ __launch_bounds__(THREADS) void norm_grad_kernel(NormGradArgs a) {
    constexpr int XB = DTypeInfo<XT>::bytes, RB = DTypeInfo<RT>::bytes;
    constexpr bool kAhead = THREADS <= 256;
    __shared__ float places[2][16];
    int turn = 0;
    const int cols = a.cols, first = threadIdx.x * 8;
    Raw<RT, THREADS, V, WHOLE> s, more;
    Raw<XT, THREADS, V, WHOLE> dy;
    float inverse = 0.0f;
    const auto load = [&](int64_t row) {
        s.load(a.s + row * a.s_stride * RB, cols);
        dy.load(a.dy + row * a.dy_stride * XB, cols);
        inverse = a.inverse[row];
        if (a.dstream) more.load(a.dstream + row * a.dstream_stride * RB, cols);
    };
    load(blockIdx.x);
    float dw[V][8];
#pragma unroll
    for (int p = 0; p < V; ++p)
#pragma unroll
        for (int k = 0; k < 8; ++k) dw[p][k] = 0.0f;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const float root = inverse;
        float n[V][8], dn[V][8], along = 0.0f;
#pragma unroll
        for (int p = 0; p < V; ++p) {
            const int c = first + p * THREADS * 8;
            float w[8];
            if (a.weight && c < cols) load_any(w, a.weight, a.weight_dtype, c, WHOLE ? 8 : cols - c);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                n[p][k] = s.value(p, k) * root;
                dn[p][k] = dy.value(p, k);
                dw[p][k] = fmaf(dn[p][k], n[p][k], dw[p][k]);
                if (a.weight) dn[p][k] *= w[k];
                if (WHOLE ? c < cols : c + k < cols) along = fmaf(dn[p][k], n[p][k], along);
            }
        }
        const int64_t next = row + gridDim.x;
        Raw<RT, THREADS, V, WHOLE> ds_in = more;
        if (kAhead && next < a.rows) load(next);
        if (a.dx || a.dresidual) {
            along = group_sum<THREADS>(along, places, turn) / (float)cols;
#pragma unroll
            for (int p = 0; p < V; ++p) {
                const int c = first + p * THREADS * 8;
                if (c >= cols) continue;
                float ds[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) ds[k] = fmaf(root, fmaf(-n[p][k], along, dn[p][k]), a.dstream ? ds_in.value(p, k) : 0.0f);
                if (a.dresidual) store_values<RT>(ds, a.dresidual + (row * cols + c) * RB, WHOLE ? 8 : cols - c);
                if (a.dx) store_values<XT>(ds, a.dx + (row * cols + c) * XB, WHOLE ? 8 : cols - c);
            }
        }
        if (!kAhead && next < a.rows) load(next);
    }
    if (a.partial) {
        float* out = a.partial + (int64_t)blockIdx.x * cols;
#pragma unroll
        for (int p = 0; p < V; ++p) {
            const int c = first + p * THREADS * 8;
            if (c < cols) store_values<DT_F32>(dw[p], out + c, WHOLE ? 8 : cols - c);
        }
    }
}

// dw: the workgroups' sums, added up in their order.  A workgroup takes 32 columns, its threads every 8th row of a column each.
constexpr int kJoinColumns = 32;
__global__ __launch_bounds__(256) void norm_join_kernel(const float* partial, int parts, int cols, char* dw, int dtype) {
    __shared__ float sums[8][kJoinColumns];
    const int column = threadIdx.x & (kJoinColumns - 1), slice = threadIdx.x / kJoinColumns, c = blockIdx.x * kJoinColumns + column;
    float sum = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int i = slice; i < parts; i += 8) sum += partial[(int64_t)i * cols + c];
    }
    sums[slice][column] = sum;
    __syncthreads();
    if (slice != 0 || c >= cols) return;
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += sums[i][column];
    if (dtype == DT_F32) reinterpret_cast<float*>(dw)[c] = sum;
    else if (dtype == DT_BF16) reinterpret_cast<__bf16*>(dw)[c] = (__bf16)sum;
    else reinterpret_cast<_Float16*>(dw)[c] = (_Float16)sum;
}

}  // namespace fo

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
namespace {
using namespace fo_host;

int validate(const char* what, int64_t rows, int64_t cols, int x_dtype, int stream_dtype, const void* weight, int weight_dtype, float eps) {
    if (rows < 0 || cols < 0) return fail(FO_ERR_INVALID_ARGUMENT, "%s: negative size", what);
    for (int dtype : {x_dtype, stream_dtype, weight ? weight_dtype : FO_F32})
        if (dtype < FO_F32 || dtype > FO_F16) return fail(FO_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    if (stream_dtype != x_dtype && stream_dtype != FO_F32) return fail(FO_ERR_UNSUPPORTED, "%s: the residual is of x's type or fp32", what);
    if (cols > FO_RMS_NORM_MOST_COLS) return fail(FO_ERR_UNSUPPORTED, "%s: rows of %lld values are too long", what, (long long)cols);
    if (rows > INT32_MAX) return fail(FO_ERR_UNSUPPORTED, "%s: %lld rows are too many", what, (long long)rows);
    if (!(eps >= 0.0f)) return fail(FO_ERR_INVALID_ARGUMENT, "%s: eps must not be negative", what);
    return 0;
}

// Calls f.template run<XT, RT>() for the types.
template <class F> int by_types(int x_dtype, int stream_dtype, const F& f) {
    if (x_dtype == FO_F32) return f.template run<fo::DT_F32, fo::DT_F32>();
    if (x_dtype == FO_BF16) return stream_dtype == FO_F32 ? f.template run<fo::DT_BF16, fo::DT_F32>() : f.template run<fo::DT_BF16, fo::DT_BF16>();
    return stream_dtype == FO_F32 ? f.template run<fo::DT_F16, fo::DT_F32>() : f.template run<fo::DT_F16, fo::DT_F16>();
}

// Threads of a workgroup and pieces of eight values that each holds: the fewest that hold a row.
template <class L> int by_width(int cols, const L& launch) {
    if (cols <= 512) return launch.template with<64, 1>();
    if (cols <= 2048) return launch.template with<256, 1>();
    if (cols <= 4096) return launch.template with<256, 2>();
    if (cols <= 8192) return launch.template with<256, 4>();
    return launch.template with<1024, 2>();
}

struct Forward {
    const fo::NormArgs& a;
    bool mx;
    hipStream_t stream;
    template <int XT, int RT> struct Width {
        const Forward& f;
        template <int THREADS, int V> int with() const {
            const int64_t most = (int64_t)compute_units() * (2048 / THREADS);
            if (most <= 0) return fail(FO_ERR_NO_DEVICE, "no device");
            const dim3 grid((unsigned)(f.a.rows < most ? f.a.rows : most)), threads(THREADS);
            const bool whole = f.a.cols % 8 == 0;
            if (f.mx && whole) fo::norm_kernel<XT, RT, THREADS, V, true, true><<<grid, threads, 0, f.stream>>>(f.a);
            else if (f.mx) fo::norm_kernel<XT, RT, THREADS, V, true, false><<<grid, threads, 0, f.stream>>>(f.a);
            else if (whole) fo::norm_kernel<XT, RT, THREADS, V, false, true><<<grid, threads, 0, f.stream>>>(f.a);
            else fo::norm_kernel<XT, RT, THREADS, V, false, false><<<grid, threads, 0, f.stream>>>(f.a);
            return check_hip(hipGetLastError(), "fo_rms_norm");
        }
    };
    template <int XT, int RT> int run() const { return by_width(a.cols, Width<XT, RT>{*this}); }
};

// Workgroups of the backward pass, each with a row of partial sums.
int64_t grad_groups(int64_t rows, int cus) { return rows < 2 * (int64_t)cus ? rows : 2 * (int64_t)cus; }

struct Backward {
    const fo::NormGradArgs& a;
    unsigned grid;
    hipStream_t stream;
    template <int XT, int RT> struct Width {
        const Backward& b;
        template <int THREADS, int V> int with() const {
            if (b.a.cols % 8 == 0) fo::norm_grad_kernel<XT, RT, THREADS, V, true><<<dim3(b.grid), dim3(THREADS), 0, b.stream>>>(b.a);
            else fo::norm_grad_kernel<XT, RT, THREADS, V, false><<<dim3(b.grid), dim3(THREADS), 0, b.stream>>>(b.a);
            return check_hip(hipGetLastError(), "fo_rms_norm_backward");
        }
    };
    template <int XT, int RT> int run() const { return by_width(a.cols, Width<XT, RT>{*this}); }
};

int forward(const char* what, const fo::NormArgs& a, int x_dtype, int stream_dtype, bool mx, void* stream) {
    if (a.rows == 0 || a.cols == 0) return 0;
    if (!a.x || !a.y || !a.residual != !a.stream) return fail(FO_ERR_INVALID_ARGUMENT, "%s: x, the result, and a stream where there is a residual must be given", what);
    return by_types(x_dtype, stream_dtype, Forward{a, mx, (hipStream_t)stream});
}

}  // namespace

extern "C" {

int fo_rms_norm(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, const void* residual, int stream_dtype, int64_t residual_stride,
                const void* weight, int weight_dtype, float eps, void* out_stream, void* y, float* inverse, void* stream) {
    if (!residual) stream_dtype = x_dtype;
    if (int rc = validate("fo_rms_norm", rows, cols, x_dtype, stream_dtype, weight, weight_dtype, eps)) return rc;
    const fo::NormArgs a{(const char*)x, (const char*)residual, (const char*)weight, (char*)out_stream, (char*)y, nullptr, inverse, x_stride, residual_stride,
                         rows, (int)cols, weight_dtype, eps};
    return forward("fo_rms_norm", a, x_dtype, stream_dtype, false, stream);
}

int fo_rms_norm_mxfp4(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, const void* residual, int stream_dtype, int64_t residual_stride,
                      const void* weight, int weight_dtype, float eps, void* out_stream, void* codes, void* scales, void* stream) {
    if (!residual) stream_dtype = x_dtype;
    if (int rc = validate("fo_rms_norm_mxfp4", rows, cols, x_dtype, stream_dtype, weight, weight_dtype, eps)) return rc;
    if (rows != 0 && cols != 0 && (!scales || (uintptr_t)codes & 15)) return fail(FO_ERR_INVALID_ARGUMENT, "scales must be given, codes aligned to 16 bytes");
    const fo::NormArgs a{(const char*)x, (const char*)residual, (const char*)weight, (char*)out_stream, (char*)codes, (uint8_t*)scales, nullptr, x_stride,
                         residual_stride, rows, (int)cols, weight_dtype, eps};
    return forward("fo_rms_norm_mxfp4", a, x_dtype, stream_dtype, true, stream);
}

int64_t fo_rms_norm_backward_workspace(int64_t rows, int64_t cols) {
    if (int rc = validate("fo_rms_norm_backward", rows, cols, FO_F32, FO_F32, nullptr, 0, 0.0f)) return rc;
    if (rows == 0 || cols == 0) return 0;
    const int cus = compute_units();
    if (cus <= 0) return fail(FO_ERR_NO_DEVICE, "no device");
    return grad_groups(rows, cus) * cols * 4;
}

int fo_rms_norm_backward(const void* s, int stream_dtype, int64_t s_stride, const void* weight, int weight_dtype, const float* inverse, const void* dy,
                         int x_dtype, int64_t dy_stride, const void* dstream, int64_t dstream_stride, int64_t rows, int64_t cols, void* dx, void* dresidual,
                         void* dw, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "fo_rms_norm_backward";
    if (int rc = validate(what, rows, cols, x_dtype, stream_dtype, weight, weight_dtype, 0.0f)) return rc;
    if (rows == 0 || cols == 0) return 0;
    if (!s || !inverse || !dy || (!dx && !dresidual && !dw)) return fail(FO_ERR_INVALID_ARGUMENT, "%s: s, inverse, dy and a result must be given", what);
    if (dw && !weight) return fail(FO_ERR_INVALID_ARGUMENT, "%s: a gradient of no weight", what);
    const int cus = compute_units();
    if (cus <= 0) return fail(FO_ERR_NO_DEVICE, "no device");
    const int64_t groups = grad_groups(rows, cus);
    if (dw && (!workspace || workspace_bytes < groups * cols * 4 || (uintptr_t)workspace & 15))
        return fail(FO_ERR_INVALID_ARGUMENT, "a workspace of %lld bytes, aligned to 16, is needed", (long long)(groups * cols * 4));
    const fo::NormGradArgs a{(const char*)s, (const char*)weight, inverse, (const char*)dy, (const char*)dstream, (char*)dx, (char*)dresidual,
                             dw ? (float*)workspace : nullptr, s_stride, dy_stride, dstream_stride, rows, (int)cols, weight_dtype};
    if (int rc = by_types(x_dtype, stream_dtype, Backward{a, (unsigned)groups, (hipStream_t)stream})) return rc;
    if (!dw) return 0;
    const unsigned grid = (unsigned)((cols + fo::kJoinColumns - 1) / fo::kJoinColumns);
    fo::norm_join_kernel<<<dim3(grid), dim3(256), 0, (hipStream_t)stream>>>((const float*)workspace, (int)groups, (int)cols, (char*)dw, weight_dtype);
    return check_hip(hipGetLastError(), what);
}

}  // extern "C"
