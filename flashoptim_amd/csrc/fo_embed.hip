// Rows of an embedding matrix by token, and the matrix's gradient.
//
//   y[i] = scale weight[tokens[i]]          dw[v] = scale (sum of dy[i] over the i with tokens[i] = v)
//
// The gradient is a sum over lists of positions, one list per row.  Positions are sorted by token, in their own order within a token, so a
// list is a run of the sorted array, and every row of dw is written once, by a sum whose order is fixed: no atomics, the
// same bits every time.
//
// Sorting.  A key is token << 32 | position, so no two are equal and a sort of keys is a stable sort of tokens.  Workgroups of 256
// threads sort runs of 512 keys, each key's place being the number of smaller ones (512 comparisons against LDS, no exchanges);
// then sixteen runs at a time are merged, again by counting: a key's place in the merged run is its place in its own plus
// the numbers of smaller keys in the fifteen others, binary searches that do not wait for one another (the first merge's in LDS).  8192 tokens take
// two launches, where the lists begin included, 131072 four.
//
// Summing.  A wavefront adds up a row's list, up to `window` positions of it.  Longer lists (padding, the most
// frequent words) are cut at multiples of that in the sorted array and their parts summed by wavefronts of their own first, in fp32, and the row's
// wavefront adds up those sums.
#include "fo_gemm.h"
#include "fo_host.h"

namespace fo {

typedef uint64_t u64;
constexpr int kRun = 512, kSortThreads = 256;    // keys a workgroup sorts
constexpr int kWays = 16;                        // runs that one merge takes
constexpr int kMergeThreads = 256;
constexpr u32 kNoToken = (1u << 23) - 1;         // sorts last; tokens are below FO_EMBEDDING_MOST_ROWS

struct Tokens {
    const void* p;
    int bytes;
    __device__ __forceinline__ int64_t operator[](int64_t i) const {
        return bytes == 8 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
    }
};

// Runs of kRun keys, sorted.  Within a run token << 9 | place is a key of 32 bits, so a 16-byte read from LDS brings four to compare with.
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(Tokens tokens, int n, int64_t vocabulary, int64_t skip, u64* keys) {
    __shared__ __attribute__((aligned(16))) u32 run[kRun];
    const int first = (int)blockIdx.x * kRun;
    u32 mine[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int at = threadIdx.x + k * kSortThreads;
        u32 t = kNoToken;
        if (first + at < n) {
            const int64_t token = tokens[first + at];
            if (token >= 0 && token < vocabulary && token != skip) t = (u32)token;
        }
        mine[k] = t << 9 | (u32)at;    // what lies behind the last token sorts behind it
        run[at] = mine[k];
    }
    __syncthreads();
    int place[2] = {0, 0};
#pragma unroll 8
    for (int i = 0; i < kRun; i += 4) {
        const u32x4 other = *reinterpret_cast<const u32x4*>(run + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            place[0] += other[e] < mine[0];
            place[1] += other[e] < mine[1];
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int at = threadIdx.x + k * kSortThreads;
        if (first + at < n) keys[first + place[k]] = (u64)(mine[k] >> 9) << 32 | (u32)(first + at);
    }
}

// How many of the sorted keys[0 .. size) are below `limit`: kWays searches at a time, each run's in its own registers, so that a step waits for memory
// once.  Steps: 2^(steps - 1) <= longest run < 2^steps.
template <class K> __device__ __forceinline__ void search_runs(const K* keys, const int (&start)[kWays], const int (&size)[kWays], int last, int steps, K limit, int (&below)[kWays]) {
    int low[kWays], left[kWays];
#pragma unroll
    for (int r = 0; r < kWays; ++r) { low[r] = start[r]; left[r] = size[r]; }
    for (int s = 0; s < steps; ++s) {
        K other[kWays];
#pragma unroll
        for (int r = 0; r < kWays; ++r) {
            const int at = low[r] + (left[r] >> 1);
            other[r] = keys[at < last ? at : last];
        }
#pragma unroll
        for (int r = 0; r < kWays; ++r) {
            const int half = left[r] >> 1;
            const bool more = left[r] > 0 && other[r] < limit;
            low[r] += more ? half + 1 : 0;
            left[r] = more ? left[r] - half - 1 : half;
        }
    }
#pragma unroll
    for (int r = 0; r < kWays; ++r) below[r] = low[r] - start[r];
}

// Runs of `length` keys in `from` become runs of kWays times as many in `to`.  A thread takes a key.
__global__ __launch_bounds__(kMergeThreads) void embed_merge_kernel(const u64* __restrict__ from, u64* __restrict__ to, int n, int length, int steps) {
    const int i = (int)blockIdx.x * kMergeThreads + threadIdx.x;
    if (i >= n) return;
    const u64 key = from[i];
    const int group = i / (length * kWays) * (length * kWays);
    int start[kWays], size[kWays], below[kWays];
#pragma unroll
    for (int r = 0; r < kWays; ++r) {
        start[r] = group + r * length;
        size[r] = start[r] >= n ? 0 : n - start[r] < length ? n - start[r] : length;
    }
    search_runs<u64>(from, start, size, n - 1, steps, key, below);
    int place = 0;
#pragma unroll
    for (int r = 0; r < kWays; ++r) place += below[r];    // its own run: its place there
    to[group + place] = key;
}

// The first merge, of runs of kRun keys, whose tokens a workgroup brings into LDS; kPer keys a thread.  Where that is all there is to merge, the workgroups
// from `merging` on write starts[v], the number of tokens below v, for v = 0 .. vocabulary.
constexpr int kMergeKeys = kRun * kWays, kPer = 2;
__global__ __launch_bounds__(kMergeThreads) void embed_first_merge_kernel(const u64* __restrict__ from, u64* __restrict__ to, int n, int merging, int64_t vocabulary, int* starts) {
    __shared__ u32 tokens[kMergeKeys];
    const bool merges = (int)blockIdx.x < merging;
    const int i0 = merges ? (int)blockIdx.x * kMergeThreads * kPer : 0, group = i0 / kMergeKeys * kMergeKeys;
    const int here = n - group < kMergeKeys ? n - group : kMergeKeys;
    for (int k = threadIdx.x; k < here; k += kMergeThreads) tokens[k] = (u32)(from[group + k] >> 32);
    __syncthreads();
    int start[kWays], size[kWays], below[kWays];
#pragma unroll
    for (int r = 0; r < kWays; ++r) {
        start[r] = r * kRun;
        size[r] = start[r] >= here ? 0 : here - start[r] < kRun ? here - start[r] : kRun;
    }
    if (!merges) {
        const int64_t v = (int64_t)((int)blockIdx.x - merging) * kMergeThreads + threadIdx.x;
        if (v > vocabulary) return;
        search_runs<u32>(tokens, start, size, here - 1, 10, (u32)v, below);
        int all = 0;
#pragma unroll
        for (int r = 0; r < kWays; ++r) all += below[r];
        starts[v] = all;
        return;
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int i = i0 + k * kMergeThreads + threadIdx.x;
        if (i >= n) return;
        const int own = (i - group) / kRun;
        const u32 token = tokens[i - group];
        // equal tokens keep the order of their runs: in those before its own they count as smaller
        int low[kWays], left[kWays];
#pragma unroll
        for (int r = 0; r < kWays; ++r) { low[r] = start[r]; left[r] = r == own ? 0 : size[r]; }
        for (int s = 0; s < 10; ++s) {
#pragma unroll
            for (int r = 0; r < kWays; ++r) {
                const int half = left[r] >> 1, at = low[r] + half;
                const u32 other = tokens[at < here ? at : here - 1];
                const bool more = left[r] > 0 && other < token + (r < own ? 1u : 0u);
                low[r] += more ? half + 1 : 0;
                left[r] = more ? left[r] - half - 1 : half;
            }
        }
        int place = i - group - own * kRun;
#pragma unroll
        for (int r = 0; r < kWays; ++r) place += r == own ? 0 : low[r] - start[r];
        to[group + place] = from[i];
    }
}

// starts[v]: the first sorted key of a token of v or more, for v = 0 .. vocabulary.
__global__ __launch_bounds__(256) void embed_starts_kernel(const u64* keys, int n, int64_t vocabulary, int* starts) {
    const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (v > vocabulary) return;
    const u64 want = (u64)v << 32;
    int low = 0, high = n;
    while (low < high) {
        const int mid = (low + high) >> 1;
        if (keys[mid] < want) low = mid + 1; else high = mid;
    }
    starts[v] = low;
}

struct EmbedGrad {
    const u64* keys;
    const int* starts;
    const char* dy;
    char* dw;
    float* partial;          // two rows per window
    int64_t dy_stride, n;
    int cols, vocabulary, window;
    float scale;
};

// Lanes take eight neighbouring values each; blockIdx.y says which 512 columns.
constexpr int kEmbedColumns = 512;

// The rows of dy that keys[first .. end) name, added up; N of them under way.
template <int DT, int N> __device__ __forceinline__ void add_rows(float (&sum)[8], const EmbedGrad& a, int64_t first, int64_t end, int c) {
    constexpr int B = DTypeInfo<DT>::bytes;
    int64_t i = first;
    for (; i + N <= end; i += N) {
        float v[N][8];
#pragma unroll
        for (int k = 0; k < N; ++k) load_values<DT>(v[k], a.dy + ((int64_t)(u32)a.keys[i + k] * a.dy_stride + c) * B, a.cols - c);
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += v[k][e];
    }
#pragma unroll 1
    for (; i < end; ++i) {
        float v[8];
        load_values<DT>(v, a.dy + ((int64_t)(u32)a.keys[i] * a.dy_stride + c) * B, a.cols - c);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += v[e];
    }
}

// Sums of the long lists' parts.  At most two lists longer than a window reach into one: the one that began before it (its part goes to row
// 2 w) and the last one that begins in it (2 w + 1).
template <int DT> __global__ __launch_bounds__(64) void embed_parts_kernel(EmbedGrad a) {
    const int64_t w = blockIdx.x, first = w * a.window, end = first + a.window < a.n ? first + a.window : a.n;
    const int c = (int)blockIdx.y * kEmbedColumns + threadIdx.x * 8;
    if (c >= a.cols) return;
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
        const u32 token = (u32)(a.keys[which ? end - 1 : first] >> 32);
        if (token >= (u32)a.vocabulary) continue;
        const int64_t start = a.starts[token], stop = a.starts[token + 1];
        if (stop - start <= a.window || (which ? start < first : start >= first)) continue;
        float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        add_rows<DT, 16>(sum, a, start > first ? start : first, stop < end ? stop : end, c);
        store_values<DT_F32>(sum, a.partial + (2 * w + which) * a.cols + c, a.cols - c);
    }
}

// A wavefront writes 512 columns of a row of dw.
template <int DT> __global__ __launch_bounds__(256) void embed_rows_kernel(EmbedGrad a) {
    constexpr int B = DTypeInfo<DT>::bytes;
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = (int)blockIdx.y * kEmbedColumns + (threadIdx.x & 63) * 8;
    if (row >= a.vocabulary || c >= a.cols) return;
    const int start = a.starts[row], stop = a.starts[row + 1];
    char* out = a.dw + (row * a.cols + c) * B;
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (stop - start > a.window) {
        const int64_t last = (stop - 1) / a.window;
        int64_t w = start / a.window;
        // the window in which the list begins, then those that it goes on into
        load_values<DT_F32>(sum, a.partial + (2 * w + 1) * a.cols + c, a.cols - c);
#pragma unroll 8
        for (++w; w <= last; ++w) {
            float v[8];
            load_values<DT_F32>(v, a.partial + 2 * w * a.cols + c, a.cols - c);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += v[e];
        }
    } else if (stop > start) {
        add_rows<DT, 4>(sum, a, start, stop, c);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] *= a.scale;
    store_values<DT>(sum, out, a.cols - c);
}

// A wavefront writes 512 columns of y's rows.
template <int DT> __global__ __launch_bounds__(256) void embed_kernel(Tokens tokens, int64_t n, const char* weight, int64_t stride, int64_t vocabulary, int cols,
                                                                      float scale, char* y) {
    constexpr int B = DTypeInfo<DT>::bytes;
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = (int)blockIdx.y * kEmbedColumns + (threadIdx.x & 63) * 8;
    if (row >= n || c >= cols) return;
    const int64_t token = tokens[row];
    float v[8];
    if (token >= 0 && token < vocabulary) {
        load_values<DT>(v, weight + (token * stride + c) * B, cols - c);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= scale;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_nanf("");
    }
    store_values<DT>(v, y + (row * cols + c) * B, cols - c);
}

}  // namespace fo

// ------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------
namespace {
using namespace fo_host;

constexpr int64_t kMostCols = 65535ll * fo::kEmbedColumns;

int validate(const char* what, int index_bytes, int64_t n, int dtype, int64_t vocabulary, int64_t cols) {
    if (n < 0 || vocabulary < 0 || cols < 0) return fail(FO_ERR_INVALID_ARGUMENT, "%s: negative size", what);
    if (index_bytes != 4 && index_bytes != 8) return fail(FO_ERR_INVALID_ARGUMENT, "%s: tokens of %d bytes", what, index_bytes);
    if (dtype < FO_F32 || dtype > FO_F16) return fail(FO_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    if (n > FO_EMBEDDING_MOST_TOKENS || vocabulary > FO_EMBEDDING_MOST_ROWS || cols > kMostCols) return fail(FO_ERR_UNSUPPORTED, "%s: too many tokens, rows or columns", what);
    return 0;
}

// At most twice as many windows as a window has positions, so that neither a list's parts nor their sums keep one wavefront long.
int window_of(int64_t n) {
    int w = 64;
    while (2 * (int64_t)w * w < n && w < 4096) w *= 2;
    return w;
}

struct Layout { int64_t keys, more, starts, partial, total; };
Layout layout(int64_t n, int64_t vocabulary, int64_t cols) {
    const auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    Layout l{};
    l.more = up(n * 8);
    l.starts = l.more + up(n * 8);
    l.partial = l.starts + up((vocabulary + 1) * 4);
    const int64_t w = window_of(n);
    l.total = l.partial + (n > w ? up((n + w - 1) / w * 2 * cols * 4) : 0);
    return l;
}

unsigned blocks(int64_t n, int64_t per) { return (unsigned)((n + per - 1) / per); }

template <int DT> int forward(const fo::Tokens& t, int64_t n, const void* weight, int64_t stride, int64_t vocabulary, int64_t cols, float scale, void* y, hipStream_t s) {
    const dim3 grid(blocks(n, 4), blocks(cols, fo::kEmbedColumns));
    fo::embed_kernel<DT><<<grid, dim3(256), 0, s>>>(t, n, (const char*)weight, stride, vocabulary, (int)cols, scale, (char*)y);
    return check_hip(hipGetLastError(), "fo_embedding");
}

template <int DT> int sums(const fo::EmbedGrad& a, hipStream_t s) {
    const unsigned across = blocks(a.cols, fo::kEmbedColumns);
    if (a.n > a.window) {
        fo::embed_parts_kernel<DT><<<dim3(blocks(a.n, a.window), across), dim3(64), 0, s>>>(a);
        if (int rc = check_hip(hipGetLastError(), "fo_embedding_backward")) return rc;
    }
    fo::embed_rows_kernel<DT><<<dim3(blocks(a.vocabulary, 4), across), dim3(256), 0, s>>>(a);
    return check_hip(hipGetLastError(), "fo_embedding_backward");
}

}  // namespace

extern "C" {

int fo_embedding(const void* tokens, int index_bytes, int64_t n_tokens, const void* weight, int dtype, int64_t vocabulary, int64_t cols, int64_t weight_stride,
                 float scale, void* y, void* stream) {
    if (int rc = validate("fo_embedding", index_bytes, n_tokens, dtype, vocabulary, cols)) return rc;
    if (n_tokens == 0 || cols == 0) return 0;
    if (!tokens || !y || (vocabulary > 0 && !weight)) return fail(FO_ERR_INVALID_ARGUMENT, "tokens, weight and y must not be NULL");
    const fo::Tokens t{tokens, index_bytes};
    switch (dtype) {
        case FO_F32: return forward<fo::DT_F32>(t, n_tokens, weight, weight_stride, vocabulary, cols, scale, y, (hipStream_t)stream);
        case FO_BF16: return forward<fo::DT_BF16>(t, n_tokens, weight, weight_stride, vocabulary, cols, scale, y, (hipStream_t)stream);
        default: return forward<fo::DT_F16>(t, n_tokens, weight, weight_stride, vocabulary, cols, scale, y, (hipStream_t)stream);
    }
}

int64_t fo_embedding_backward_workspace(int64_t n_tokens, int64_t vocabulary, int64_t cols) {
    if (int rc = validate("fo_embedding_backward", 8, n_tokens, FO_F32, vocabulary, cols)) return rc;
    return layout(n_tokens, vocabulary, cols).total;
}

int fo_embedding_backward(const void* tokens, int index_bytes, int64_t n_tokens, const void* dy, int dtype, int64_t dy_stride, int64_t vocabulary, int64_t cols,
                          float scale, int64_t padding, void* dw, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "fo_embedding_backward";
    if (int rc = validate(what, index_bytes, n_tokens, dtype, vocabulary, cols)) return rc;
    if (vocabulary == 0 || cols == 0) return 0;
    const Layout l = layout(n_tokens, vocabulary, cols);
    if (!dw || (n_tokens > 0 && (!tokens || !dy))) return fail(FO_ERR_INVALID_ARGUMENT, "%s: tokens, dy and dw must not be NULL", what);
    if (!workspace || workspace_bytes < l.total || (uintptr_t)workspace & 255)
        return fail(FO_ERR_INVALID_ARGUMENT, "a workspace of %lld bytes, aligned to 256, is needed", (long long)l.total);
    const hipStream_t s = (hipStream_t)stream;
    char* base = (char*)workspace;
    fo::u64 *keys = (fo::u64*)base, *other = (fo::u64*)(base + l.more);
    int* starts = (int*)(base + l.starts);
    const int n = (int)n_tokens;
    const unsigned starting = blocks(vocabulary + 1, 256);
    if (n <= fo::kMergeKeys && n > 0) {
        fo::embed_sort_kernel<<<dim3(blocks(n, fo::kRun)), dim3(fo::kSortThreads), 0, s>>>(fo::Tokens{tokens, index_bytes}, n, vocabulary, padding, other);
        if (int rc = check_hip(hipGetLastError(), what)) return rc;
        const unsigned merging = blocks(n, fo::kMergeThreads * fo::kPer);
        fo::embed_first_merge_kernel<<<dim3(merging + starting), dim3(fo::kMergeThreads), 0, s>>>(other, keys, n, (int)merging, vocabulary, starts);
        if (int rc = check_hip(hipGetLastError(), what)) return rc;
    } else {
        // where the keys are to end up decides where they begin
        int merges = 0;
        for (int64_t length = fo::kRun; length < n; length *= fo::kWays) ++merges;
        fo::u64 *from = merges & 1 ? other : keys, *to = merges & 1 ? keys : other;
        if (n > 0) {
            fo::embed_sort_kernel<<<dim3(blocks(n, fo::kRun)), dim3(fo::kSortThreads), 0, s>>>(fo::Tokens{tokens, index_bytes}, n, vocabulary, padding, from);
            if (int rc = check_hip(hipGetLastError(), what)) return rc;
        }
        int steps = 10;    // of a search among `length` keys
        for (int64_t length = fo::kRun; length < n; length *= fo::kWays, steps += 4) {
            if (length == fo::kRun) fo::embed_first_merge_kernel<<<dim3(blocks(n, fo::kMergeThreads * fo::kPer)), dim3(fo::kMergeThreads), 0, s>>>(from, to, n, INT32_MAX, 0, nullptr);
            else fo::embed_merge_kernel<<<dim3(blocks(n, fo::kMergeThreads)), dim3(fo::kMergeThreads), 0, s>>>(from, to, n, (int)length, steps);
            if (int rc = check_hip(hipGetLastError(), what)) return rc;
            fo::u64* t = from; from = to; to = t;
        }
        fo::embed_starts_kernel<<<dim3(starting), dim3(256), 0, s>>>(keys, n, vocabulary, starts);
        if (int rc = check_hip(hipGetLastError(), what)) return rc;
    }
    const fo::EmbedGrad a{keys, starts, (const char*)dy, (char*)dw, (float*)(base + l.partial), dy_stride, n_tokens, (int)cols, (int)vocabulary, window_of(n_tokens), scale};
    switch (dtype) {
        case FO_F32: return sums<fo::DT_F32>(a, s);
        case FO_BF16: return sums<fo::DT_BF16>(a, s);
        default: return sums<fo::DT_F16>(a, s);
    }
}

}  // extern "C"
