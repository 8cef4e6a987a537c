// Rows of an embedding matrix by token, and the matrix's gradient.
//
//   y[i] = scale weight[tokens[i]]          dw[v] = scale (sum of dy[i] over the i with tokens[i] = v)
//
// The gradient is a sum over lists of positions, one list per row.  dw is filled with zeros, positions are sorted by token, in their own order within a
// token, so a list is a run of the sorted array, and every row that has a list is written once more, by a sum whose order is fixed: no atomics,
// the same bits every time.
//
// Sorting.  A key is token << 32 | position, so no two are equal and a sort of keys is a stable sort of tokens.  A key's place is the
// number of keys below it, counted: in the 64 of its wavefront by comparing with each, in the workgroup's eight such runs by binary searches
// in LDS, that makes runs of 512; then in sixteen of those at a time, again by binary searches, the first time in LDS, from 131072 tokens on in
// memory.  None of these launches has work for a fill's memory bandwidth, so the first two carry the fill with them: 128256 x 4096 bf16 in 72 + 89 us (6.5 TB/s), the
// sorting of 8192 tokens in their shadow (4 + 4 us for 1003 tokens and a small matrix).
//
// Summing.  The sorted array is cut into windows of the same length whatever the lists, a wavefront takes a window (and 512 columns), so the
// padding token or the most frequent word keeps nobody longer than the others.  A list that ends where its window does not is complete;
// lists that go on over a border leave fp32 sums, which another launch adds up.
#include "fo_gemm.h"
#include "fo_host.h"

namespace fo {

typedef uint64_t u64;
constexpr int kRun = 512;                        // keys, and threads, of a workgroup that sorts
constexpr int kWays = 16;                        // runs that one merge takes
constexpr int kMergeKeys = kRun * kWays, kMergeThreads = 256;
constexpr u32 kNoToken = (1u << 23) - 1;         // sorts last; tokens are below it, FO_EMBEDDING_MOST_ROWS
constexpr int kFillBytes = 65536;                // a workgroup's share of a fill

struct Tokens {
    const void* p;
    int bytes;
    __device__ __forceinline__ int64_t operator[](int64_t i) const {
        return bytes == 8 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
    }
};

// Zeros from `first` of kFillBytes on.
template <int THREADS> __device__ __forceinline__ void fill(char* to, int64_t bytes, int64_t first) {
    const int64_t from = first * kFillBytes;
    const u32x4 zero = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < kFillBytes / 16 / THREADS; ++k) {
        const int64_t at = from + ((int64_t)k * THREADS + threadIdx.x) * 16;
        if (at + 16 <= bytes) *reinterpret_cast<FO_GLOBAL u32x4_any*>((FO_GLOBAL char*)to + at) = zero;
        else for (int64_t i = at; i < bytes; ++i) to[i] = 0;
    }
}

// The number of the run's 2^log keys below `limit`; LDS holds kNoToken << 9 and more behind the last key.  `key(i)` is its i-th.
template <int LOG, class F> __device__ __forceinline__ int below(u32 limit, const F& key) {
    int pos = 0;
#pragma unroll
    for (int step = 1 << (LOG - 1); step > 0; step >>= 1) pos += key(pos + step - 1) < limit ? step : 0;
    return pos + (key(pos) < limit ? 1 : 0);
}

// Runs of kRun keys, sorted; workgroups from `sorting` on fill.  Within a run token << 9 | place is a key of 32 bits.
__global__ __launch_bounds__(kRun) void embed_sort_kernel(Tokens tokens, int n, int64_t vocabulary, int64_t skip, u64* keys, int sorting, char* filled, int64_t fill_bytes) {
    if ((int)blockIdx.x >= sorting) { fill<kRun>(filled, fill_bytes, (int64_t)blockIdx.x - sorting); return; }
    __shared__ u32 run[kRun];
    const int first = (int)blockIdx.x * kRun, at = threadIdx.x, wave = at >> 6;
    u32 t = kNoToken;
    if (first + at < n) {
        const int64_t token = tokens[first + at];
        if (token >= 0 && token < vocabulary && token != skip) t = (u32)token;
    }
    const u32 mine = t << 9 | (u32)at;    // what lies behind the last token sorts behind it
    int place = 0;
#pragma unroll
    for (int i = 0; i < 64; ++i) place += (u32)__builtin_amdgcn_readlane((int)mine, i) < mine;
    run[wave * 64 + place] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kRun / 64; ++w) {
        const int there = below<6>(mine, [&](int i) { return run[w * 64 + i]; });
        place += w == wave ? 0 : there;
    }
    if (first + at < n) keys[first + place] = (u64)t << 32 | (u32)(first + at);
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

// The first merge, of runs of kRun keys, whose tokens a workgroup brings into LDS; workgroups from `merging` on fill, beginning with `first_fill`.
__global__ __launch_bounds__(kMergeThreads) void embed_first_merge_kernel(const u64* __restrict__ from, u64* __restrict__ to, int n, int merging, char* filled, int64_t fill_bytes,
                                                                          int64_t first_fill) {
    if ((int)blockIdx.x >= merging) { fill<kMergeThreads>(filled, fill_bytes, first_fill + (int64_t)blockIdx.x - merging); return; }
    __shared__ u32 tokens[kMergeKeys];
    const int i = (int)blockIdx.x * kMergeThreads + threadIdx.x, group = i / kMergeKeys * kMergeKeys;
    const int here = n - group < kMergeKeys ? n - group : kMergeKeys, runs = (here + kRun - 1) / kRun;
#pragma unroll 4
    for (int k = threadIdx.x; k < runs * kRun; k += kMergeThreads) tokens[k] = k < here ? (u32)(from[group + k] >> 32) : ~0u;
    __syncthreads();
    if (i >= n) return;
    const int own = (i - group) / kRun;
    const u32 token = tokens[i - group];
    int place = i - group - own * kRun;
#pragma unroll
    for (int r = 0; r < kWays; ++r) {
        if (r >= runs) break;
        // equal tokens keep the order of their runs: those of runs before its own count as below it
        const int there = below<9>(token + (r < own ? 1u : 0u), [&](int k) { return tokens[r * kRun + k]; });
        place += r == own ? 0 : there;
    }
    to[group + place] = from[i];
}

struct EmbedGrad {
    const u64* keys;         // sorted
    const char* dy;
    char* dw;
    float* partial;          // two rows per window: of the list that comes into it, of the one that begins in it and goes on
    int64_t dy_stride;
    int n, cols, window;
    float scale;
    __device__ __forceinline__ u32 token(int i) const { return (u32)(keys[i] >> 32); }
    __device__ __forceinline__ float* part(int w, int which, int c) const { return partial + (2 * (int64_t)w + which) * cols + c; }
};

// Lanes take eight neighbouring values each; blockIdx.y says which 512 columns.
constexpr int kEmbedColumns = 512;

template <int DT> __device__ __forceinline__ void store_row(const EmbedGrad& a, u32 token, int c, const float (&sum)[8]) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = sum[e] * a.scale;
    store_values<DT>(v, a.dw + ((int64_t)token * a.cols + c) * DTypeInfo<DT>::bytes, a.cols - c);
}

// A lane's part of kAtOnce rows of dy, as it comes from memory.
constexpr int kAtOnce = 8;
template <int DT> struct SomeRows {
    static constexpr int B = DTypeInfo<DT>::bytes, EPL = 16 / B;
    Pack<B, EPL> d[kAtOnce][8 / EPL];
    // Of the positions that lanes `at` on of the wavefront hold, those before `end`.
    __device__ __forceinline__ void load(const EmbedGrad& a, u32 positions, int at, int end, int c) {
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {
            if (at + k >= end) break;
            const u32 position = (u32)__builtin_amdgcn_readlane((int)positions, at + k);
            const char* row = a.dy + ((int64_t)position * a.dy_stride + c) * B;
#pragma unroll
            for (int part = 0; part < 8 / EPL; ++part) load_piece<B, EPL>(d[k][part], row + part * 16, a.cols - c - part * EPL);
        }
    }
    __device__ __forceinline__ float value(int k, int e) const { return widen<DT, EPL>(d[k][e / EPL], e % EPL); }
};

// A wavefront adds up the lists, and parts of lists, of its window.  Its lanes hold 64 keys at a time, so that only rows of dy are waited for, kAtOnce of them while the
// kAtOnce before are added: 8192 rows of 4096 bf16 values in 37 us (3.5 TB/s read and written; 41 with keys read as they are needed).
template <int DT> __global__ __launch_bounds__(256) void embed_windows_kernel(EmbedGrad a) {
    const int w = (int)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int c = (int)blockIdx.y * kEmbedColumns + lane * 8;
    const int first = w * a.window, end = first + a.window < a.n ? first + a.window : a.n;
    if (first >= a.n) return;
    const bool mine = c < a.cols;
    const u32 before = first > 0 ? a.token(first - 1) : kNoToken;
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    bool came_in = false;
    for (int chunk = first; chunk < end; chunk += 64) {
        const int here = end - chunk < 64 ? end - chunk : 64;
        const u64 key = a.keys[chunk + lane < a.n ? chunk + lane : a.n - 1];
        const u32 behind = chunk + here < a.n ? a.token(chunk + here) : kNoToken;
        const u32 tokens = (u32)(key >> 32), positions = (u32)key;
        u32 token = (u32)__builtin_amdgcn_readlane((int)tokens, 0);
        if (chunk == first) came_in = before == token && first > 0;
        SomeRows<DT> rows, more;
        if (mine) rows.load(a, positions, 0, here, c);
        for (int i = 0; i < here; i += kAtOnce) {
            if (mine) more.load(a, positions, i + kAtOnce, here, c);
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                if (i + k >= here) break;
                if (token == kNoToken) return;    // there are none behind
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += rows.value(k, e);
                const u32 next = i + k + 1 < here ? (u32)__builtin_amdgcn_readlane((int)tokens, i + k + 1) : behind;
                if (next != token) {
                    if (mine) {
                        if (came_in) store_values<DT_F32>(sum, a.part(w, 0, c), a.cols - c);
                        else store_row<DT>(a, token, c, sum);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum[e] = 0.0f;
                    came_in = false;
                    token = next;
                } else if (chunk + i + k + 1 == end) {
                    if (mine) store_values<DT_F32>(sum, a.part(w, came_in ? 0 : 1, c), a.cols - c);
                }
            }
            rows = more;
        }
    }
}

// The list that begins in window blockIdx.x and goes on: its parts are added up, every fourth by a wavefront, and the four sums then.
template <int DT> __global__ __launch_bounds__(256) void embed_borders_kernel(EmbedGrad a) {
    __shared__ float sums[3][64][9];
    const int w = blockIdx.x, first = w * a.window, end = first + a.window;
    if (end >= a.n) return;
    const u32 token = a.token(end - 1);
    if (token == kNoToken || a.token(end) != token || (first > 0 && a.token(first) == token && a.token(first - 1) == token)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = (int)blockIdx.y * kEmbedColumns + lane * 8;
    int last = w;    // the last window that the list reaches into
    for (;;) {
        const int64_t at = (int64_t)(last + 1 + lane) * a.window;
        const uint64_t in = __builtin_amdgcn_ballot_w64(at < a.n && a.token(at < a.n ? (int)at : 0) == token);
        const int more = in == ~0ull ? 64 : __builtin_ctzll(~in);
        last += more;
        if (more < 64) break;
    }
    float sum[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (c < a.cols) {
        if (wave == 0) load_values<DT_F32>(sum, a.part(w, 1, c), a.cols - c);
#pragma unroll 8
        for (int j = w + 1 + wave; j <= last; j += 4) {
            float v[8];
            load_values<DT_F32>(v, a.part(j, 0, c), a.cols - c);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += v[e];
        }
    }
    if (wave > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[wave - 1][lane][e] = sum[e];
    }
    __syncthreads();
    if (wave > 0 || c >= a.cols) return;
#pragma unroll
    for (int q = 0; q < 3; ++q)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += sums[q][lane][e];
    store_row<DT>(a, token, c, sum);
}

// A wavefront writes 512 columns of y's rows.  Bound by memory: 8192 rows of 4096 bf16 values in 28 us (4.8 TB/s).
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
    // fewer than 2^32 threads fill
    if (n > FO_EMBEDDING_MOST_TOKENS || vocabulary > FO_EMBEDDING_MOST_ROWS || cols > kMostCols || vocabulary * cols > (int64_t)1 << 37) return fail(FO_ERR_UNSUPPORTED, "%s: too many tokens, rows or columns", what);
    return 0;
}

// At most 1024 windows of at least 16 positions, so that neither a window nor the parts of one list keep a workgroup long; at most 4096 positions.
int window_of(int64_t n) {
    int w = 16;
    while ((int64_t)w * 1024 < n && w < 4096) w *= 2;
    return w;
}

struct Layout { int64_t keys, more, partial, total; };
Layout layout(int64_t n, int64_t cols) {
    const auto up = [](int64_t b) { return (b + 255) / 256 * 256; };
    Layout l{};
    l.more = up(n * 8);
    l.partial = l.more + (n > fo::kRun ? up(n * 8) : 0);
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
    const unsigned across = blocks(a.cols, fo::kEmbedColumns), windows = blocks(a.n, a.window);
    fo::embed_windows_kernel<DT><<<dim3((windows + 3) / 4, across), dim3(256), 0, s>>>(a);
    if (int rc = check_hip(hipGetLastError(), "fo_embedding_backward")) return rc;
    if (windows == 1) return 0;
    fo::embed_borders_kernel<DT><<<dim3(windows - 1, across), dim3(256), 0, s>>>(a);
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
    return layout(n_tokens, cols).total;
}

int fo_embedding_backward(const void* tokens, int index_bytes, int64_t n_tokens, const void* dy, int dtype, int64_t dy_stride, int64_t vocabulary, int64_t cols,
                          float scale, int64_t padding, void* dw, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* what = "fo_embedding_backward";
    if (int rc = validate(what, index_bytes, n_tokens, dtype, vocabulary, cols)) return rc;
    if (vocabulary == 0 || cols == 0) return 0;
    const Layout l = layout(n_tokens, cols);
    if (!dw || (n_tokens > 0 && (!tokens || !dy))) return fail(FO_ERR_INVALID_ARGUMENT, "%s: tokens, dy and dw must not be NULL", what);
    if (n_tokens > 0 && (!workspace || workspace_bytes < l.total || (uintptr_t)workspace & 255))
        return fail(FO_ERR_INVALID_ARGUMENT, "a workspace of %lld bytes, aligned to 256, is needed", (long long)l.total);
    const hipStream_t s = (hipStream_t)stream;
    char* base = (char*)workspace;
    fo::u64 *keys = (fo::u64*)base, *other = (fo::u64*)(base + l.more);
    const int n = (int)n_tokens;
    // an odd number of merges ends in the other array
    int merges = 0;
    for (int64_t length = fo::kRun; length < n; length *= fo::kWays) ++merges;
    fo::u64 *from = merges & 1 ? other : keys, *to = merges & 1 ? keys : other;
    const int64_t bytes = vocabulary * cols * (dtype == FO_F32 ? 4 : 2), fills = (bytes + fo::kFillBytes - 1) / fo::kFillBytes, fills_first = merges > 0 ? fills / 2 : fills;
    const unsigned sorting = blocks(n, fo::kRun), merging = blocks(n, fo::kMergeThreads);
    fo::embed_sort_kernel<<<dim3(sorting + (unsigned)fills_first), dim3(fo::kRun), 0, s>>>(fo::Tokens{tokens, index_bytes}, n, vocabulary, padding, from, (int)sorting, (char*)dw, bytes);
    if (int rc = check_hip(hipGetLastError(), what)) return rc;
    if (n == 0) return 0;
    int steps = 10;    // of a search among `length` keys
    for (int64_t length = fo::kRun; length < n; length *= fo::kWays, steps += 4) {
        if (length == fo::kRun)
            fo::embed_first_merge_kernel<<<dim3(merging + (unsigned)(fills - fills_first)), dim3(fo::kMergeThreads), 0, s>>>(from, to, n, (int)merging, (char*)dw, bytes, fills_first);
        else
            fo::embed_merge_kernel<<<dim3(merging), dim3(fo::kMergeThreads), 0, s>>>(from, to, n, (int)length, steps);
        if (int rc = check_hip(hipGetLastError(), what)) return rc;
        fo::u64* t = from; from = to; to = t;
    }
    const fo::EmbedGrad a{keys, (const char*)dy, (char*)dw, (float*)(base + l.partial), dy_stride, n, (int)cols, window_of(n), scale};
    switch (dtype) {
        case FO_F32: return sums<fo::DT_F32>(a, s);
        case FO_BF16: return sums<fo::DT_BF16>(a, s);
        default: return sums<fo::DT_F16>(a, s);
    }
}

}  // extern "C"
