// Matrix product core of the gfx950 kernels that multiply: C[i][j] = sum_k A[i][k] * B[j][k], both operands with k
// contiguous, fp32 accumulation in the matrix cores.  The Newton-Schulz kernels (fo_muon.hip) run it on fp16 operands, the
// microscaled 4-bit product (fo_mx.hip) on E2M1 codes with one E8M0 scale per 32 of them.  The two differ in the matrix
// instruction only: either way a lane's operand of one 16x16 instruction is 16 bytes of one row, so a tile is rows of
// bytes and the same staging serves both.
//
// Shape.  A workgroup is four wavefronts in a 2x2 arrangement; a wavefront owns a WT x WT piece of the tile (WT = 128, 96,
// 64 or 32) and keeps it in its accumulators.  The operands pass through LDS in stages of 128 bytes of every row (64 fp16
// values, 256 codes), two stages in turn (or three or four, see below).  With WT = 128 the workgroup holds 128 KiB of LDS, a wavefront 256 accumulator
// registers and both halves of a stage's operands in registers, and one wavefront runs on each SIMD: every LDS byte read is
// used for eight instructions, which is what keeps LDS (128 bytes a clock) behind the matrix cores.
//
// Flow.  Per stage two phases of (WT/16)^2 matrix instructions.  Phase 1 multiplies the first half of the stage out of
// registers while the second half is read from LDS; then the workgroup meets (nobody reads this stage any more, and the next
// one has arrived); phase 2 multiplies the second half while the next stage's first half is read and the loads of the
// stage after it are issued into the buffer that has become free.  A load has one whole stage of multiplications to arrive; of
// 64 x 64 tiles, whose stages are short, that covers it where four or five workgroups share a compute unit.  Where one has it alone, four
// stages in LDS give a load three: 1000 x 1000 through five Newton-Schulz steps takes 148 instead of 191 us.  192 x 192 tiles have room for
// three: 14336 x 4096 takes 3.48 ms, 3.56 with two.
//
// Loads go from memory straight into LDS (16 bytes a lane, no registers).  They are inline asm: the compiler would wait for
// all of them before every LDS read.  They have no register result, and every wait for them is written out below.
//
// LDS layout: rows of 128 bytes, the eight 16-byte pieces of row r stored in the order piece ^ (r / 2 & 7).  The hardware serves a
// 16-byte read in four turns over all 64 banks, and what it takes together are not the 16 rows of one piece but eight of one and
// eight of the next: the order keeps those apart where the two pieces are neighbours, so a lane's group takes piece `group` in one phase
// and `group` + 4 in the other (bank conflicts of S of 14336 x 4096: 1.1e6 cycles; 22.9e6 with pieces 2 group and 2 group + 1, or with
// r & 7; 1000 x 1000 in all took 5 % less).  Scaled operands keep 2 group and 2 group + 1, a lane's two scales are neighbours then, and
// their conflicts are hidden: an order without them took as long.
// The order is applied to the address that a lane loads from.
//
// Either operand (not codes) may lie the other way round in memory, the contracted axis down the rows: A[k][i], B[k][j] with i and j adjacent (KA, KB).  Its stage
// is then 64 rows (32 of fp32) of a tile's width, of the same number of bytes.  The operand of a 16-bit instruction comes out of LDS through two transposing reads: sixteen
// lanes read four rows of sixteen values and get four values of a column each; fp32 ones are read value by value, which is as they are wanted.  Sixteen values of a
// row are a piece; row k keeps its pieces shifted by turned_shift(k), so that the rows that a wavefront reads at a time lie in all banks.  Rows need not be
// filled up to whole stages: those behind the last are read as copies of it, the other operand holds zeros for them.
#pragma once

#include "fo_device.h"

namespace fo {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Pieces of rows that begin at any element: global memory takes vector accesses at any address (the compiler emits them as
// such for its default unaligned access mode), so rows of odd lengths need no path of their own.
typedef u32x4 u32x4_any __attribute__((aligned(1)));
typedef u32x2 u32x2_any __attribute__((aligned(1)));

// EPL elements of EB bytes at p, `valid` of them there; the rest reads as zero and is not written.
template <int EB, int EPL> __device__ __forceinline__ void load_piece(Pack<EB, EPL>& d, const void* p, int valid) {
    if constexpr (EB > 0) {
        if (valid < EPL) { load_guarded<EB, EPL>(d, p, 0, valid); return; }
        if constexpr (EB * EPL == 16) {
            const u32x4 v = *reinterpret_cast<const FO_GLOBAL u32x4_any*>((const FO_GLOBAL char*)p);
            d.w[0] = v.x; d.w[1] = v.y; d.w[2] = v.z; d.w[3] = v.w;
        } else {
            static_assert(EB * EPL == 8, "8 or 16 bytes");
            const u32x2 v = *reinterpret_cast<const FO_GLOBAL u32x2_any*>((const FO_GLOBAL char*)p);
            d.w[0] = v.x; d.w[1] = v.y;
        }
    }
}
template <int EB, int EPL> __device__ __forceinline__ void store_piece(const Pack<EB, EPL>& d, void* p, int valid) {
    if constexpr (EB > 0) {
        if (valid < EPL) { store_guarded<EB, EPL>(d, p, 0, valid); return; }
        if constexpr (EB * EPL == 16) {
            *reinterpret_cast<FO_GLOBAL u32x4_any*>((FO_GLOBAL char*)p) = u32x4{d.w[0], d.w[1], d.w[2], d.w[3]};
        } else {
            static_assert(EB * EPL == 8, "8 or 16 bytes");
            *reinterpret_cast<FO_GLOBAL u32x2_any*>((FO_GLOBAL char*)p) = u32x2{d.w[0], d.w[1]};
        }
    }
}
// Eight values from a row of type DT, the first `valid` of them there (the others read as zero).
template <int DT> __device__ __forceinline__ void load_values(float (&v)[8], const void* p, int valid) {
    constexpr int B = DTypeInfo<DT>::bytes, EPL = 16 / B;
#pragma unroll
    for (int part = 0; part < 8 / EPL; ++part) {
        Pack<B, EPL> d;
        load_piece<B, EPL>(d, (const char*)p + part * 16, valid - part * EPL);
#pragma unroll
        for (int k = 0; k < EPL; ++k) v[part * EPL + k] = widen<DT, EPL>(d, k);
    }
}
// Eight values as a piece of a row of type DT.
template <int DT> __device__ __forceinline__ void store_values(const float (&v)[8], void* p, int valid) {
    constexpr int B = DTypeInfo<DT>::bytes, EPL = 16 / B;
#pragma unroll
    for (int part = 0; part < 8 / EPL; ++part) {
        Pack<B, EPL> d;
#pragma unroll
        for (int k = 0; k < EPL; k += 2) { float x, y; narrow_pair<DT, EPL>(d, k, v[part * EPL + k], v[part * EPL + k + 1], x, y); }
        store_piece<B, EPL>(d, (char*)p + part * 16, valid - part * EPL);
    }
}

constexpr int kStageBytes = 128;   // of each row
constexpr int kHalfBytes = 64;     // what one phase multiplies; rows are whole multiples of it

// One operand: `rows` rows of `row_bytes` (a multiple of 64), `stride` bytes apart.  Rows beyond the last are read as copies of
// the last one; what they contribute to is not stored.  scales (4-bit operands): one byte per 16 bytes of the row.
struct Operand {
    const char* data;
    int64_t stride;
    const uint8_t* scales;
    int64_t scale_stride;
    int rows;
    int depth;              // turned operands: how many rows there are along the contracted axis; `rows`, a multiple of 8, is how long they are
    int64_t part_stride;    // products in parts: bytes from a part of the values to the next
    u32 order;              // and which part each segment of the contraction takes, two bits each
    int pieces;             // 16-byte pieces of a row that there are, where it is not filled up (0: it is); the others are read as copies of the last one, and the
                            // other operand holds zeros for them
};

// The matrix instructions are inline asm so that an accumulator stays in the registers it is in (the compiler's own form lets
// result and addend differ, and with 256 accumulator registers out of 256 it spills).  What the hazard recogniser then does
// not see: an accumulator may be read by other instructions 18 wait states after the last instruction that wrote it, see
// multiply().  Results feed the next instruction on the same accumulator without a wait, at least three others lie between.
struct F16Product {
    static constexpr bool kScaled = false, kParts = false;
    static constexpr int kBytes = 2;
    typedef f16x8 Frag;
    template <int HALF> __device__ __forceinline__ static void multiply(const Frag& a, const Frag& b, f32x4& c, int, int) {
        asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    }
};

struct Bf16Product {
    static constexpr bool kScaled = false, kParts = false;
    static constexpr int kBytes = 2;
    typedef bf16x8 Frag;
    template <int HALF> __device__ __forceinline__ static void multiply(const Frag& a, const Frag& b, f32x4& c, int, int) {
        asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
    }
};

// fp32 values on the matrix cores' fp32 instructions, a sixteenth of the 16-bit rate: a lane's 16 bytes are one value for each of four instructions.  An instruction adds four
// products, so a sum of thousands is rounded often enough to show (one token's loss over 2195 values was off by 9e-6 of itself, by 1e-6 in sums of another order): every
// four stages (128 values) the sums are added to a second set, in vector registers, and begin anew.  That is 5 % of the time (512 x 1000 over 5003: 220 -> 230 us).
struct F32Product {
    static constexpr bool kScaled = false, kParts = false;
    static constexpr int kBytes = 4;
    typedef f32x4 Frag;
    template <int HALF> __device__ __forceinline__ static void multiply(const Frag& a, const Frag& b, f32x4& c, int, int) {
#pragma unroll
        for (int k = 0; k < 4; ++k) asm("v_mfma_f32_16x16x4_f32 %0, %1, %2, %0" : "+a"(c) : "v"(a[k]), "v"(b[k]));
    }
};

// Values in three bf16 parts each, part after part in memory: the contraction is kSegments products of parts one after the other, each over whole stages.
struct Bf16PartsProduct : Bf16Product {
    static constexpr bool kParts = true;
};
constexpr int kSegments = 6;

// HALF: which byte of the two scales is meant.
struct Mx4Product {
    static constexpr bool kScaled = true, kParts = false;
    static constexpr int kBytes = 2;    // of no meaning: two values to a byte
    typedef i32x4 Frag;
    template <int HALF> __device__ __forceinline__ static void multiply(const Frag& a, const Frag& b, f32x4& c, int a_scales, int b_scales) {
        if constexpr (HALF == 0)
            asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[0,0,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                : "+a"(c) : "v"(a), "v"(b), "v"(a_scales), "v"(b_scales));
        else
            asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                : "+a"(c) : "v"(a), "v"(b), "v"(a_scales), "v"(b_scales));
    }
};

// 64 lanes x 16 (4) bytes from base + lane offset to LDS at `lds` + 16 (4) * lane.  m0, which holds that address, is a reserved
// register: the compiler keeps no value in it, and nothing else in a kernel that multiplies uses it.
__device__ __forceinline__ void load_to_lds16(unsigned lds, unsigned offset, const char* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void load_to_lds4(unsigned lds, unsigned offset, const char* base) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory");
}
template <int N> __device__ __forceinline__ void wait_loads_and_lds() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory"); }
__device__ __forceinline__ void meet() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
__device__ __forceinline__ const char* uniform(const char* p) {
    const uint64_t v = (uint64_t)p;
    const u32 lo = __builtin_amdgcn_readfirstlane((u32)v), hi = __builtin_amdgcn_readfirstlane((u32)(v >> 32));
    return (const char*)(((uint64_t)hi << 32) | lo);
}

template <class Product, int WT, int STAGES, bool KA = false, bool KB = false> struct GemmTile {
    static constexpr int kStages = STAGES;        // in LDS, 2 to 4
    static constexpr int kTile = 2 * WT;          // rows and columns of a workgroup's tile
    static constexpr int kFrags = WT / 16;        // 16-row pieces of a wavefront's operands
    static constexpr int kRows = 2 * kTile;       // rows of a stage, A's then B's
    static constexpr int kScaleOffset = kRows * kStageBytes;
    static constexpr int kBuffer = kScaleOffset + (Product::kScaled ? kRows * 8 : 0);
    static constexpr int kRowLoads = kRows / 8 / 4;                          // loads of a wavefront per stage: 8 rows each
    static constexpr int kScaleLoads = Product::kScaled ? kRows / 32 / 4 : 0;   // 32 rows each
    static constexpr int kLoads = kRowLoads + kScaleLoads;
    // the epilogue moves the tile through LDS in strips of 32 rows of a wavefront, 4 floats of padding per row
    static constexpr int kStripStride = WT + 4;
    static constexpr int kStripBytes = 32 * kStripStride * 4;
    static_assert(kStages * kBuffer <= 163840 && (kStages - 1) * kLoads <= 63, "what LDS holds, what the counter of loads under way counts to");
    static constexpr int kLds = kStages * kBuffer > 4 * kStripBytes ? kStages * kBuffer : 4 * kStripBytes;

    static constexpr int kPieces = kTile / 16;    // of sixteen values, in a stage row of a turned operand
    static constexpr int kElement = Product::kBytes, kTurnedRow = kElement * kTile, kTurnedRows = kStageBytes / kElement;
    static_assert(!Product::kScaled || (!KA && !KB), "codes have no transposing read");

    typedef typename Product::Frag Frag;

    static constexpr bool kTwoSums = Product::kBytes == 4;
    static constexpr int kFlushStages = 4;

    f32x4 acc[kFrags][kFrags];
    f32x4 total[kTwoSums ? kFrags : 1][kTwoSums ? kFrags : 1];
    int first_stage = 0;       // where along the contraction this product begins
    int segment_stages = 0;    // products in parts: stages of a segment
    char* smem;
    unsigned smem_address;
    int wave, lane;

    __device__ __forceinline__ GemmTile(char* lds)
        : smem(lds), smem_address(lds_address(lds)), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), lane(threadIdx.x & 63) {}

    // ------------------------------------------------------------------------------------------- staging
    __device__ __forceinline__ static int buffer_of(int stage) { return (kStages == 3 ? stage % 3 : stage & (kStages - 1)) * kBuffer; }
    __device__ __forceinline__ static int place_of(int row) { return (row >> 1) & 7; }
    __device__ __forceinline__ static int turned_shift(int k) {
        if constexpr (kElement == 4) return k >> 2 & 3;
        return kPieces % 8 == 0 ? (k & 3) | (k >> 3 & 1) << 2 : (k >> 1 & 1) | (k >> 3 & 1) << 1;
    }
    static constexpr bool kShiftByXor = kElement == 4 || kPieces % 8 == 0;
    // Where piece `at` of stage row k lies in that row.
    __device__ __forceinline__ static int turned_place(int at, int k) {
        if constexpr (kShiftByXor) return at ^ turned_shift(k);
        const int place = at + turned_shift(k);
        return place < kPieces ? place : place - kPieces;
    }
    __device__ __forceinline__ static int turned_piece(int place, int k) {    // and back
        if constexpr (kShiftByXor) return place ^ turned_shift(k);
        const int at = place - turned_shift(k);
        return at < 0 ? at + kPieces : at;
    }
    struct Loader {
        unsigned row[kRowLoads];
        bool turned;
        int64_t part_stride;
        u32 order;
        int64_t step;            // bytes from a stage to the next
        unsigned line;           // turned: bytes from a row to the next, and the rows that there are
        int depth;
        unsigned scale[kScaleLoads > 0 ? kScaleLoads : 1];
        int piece;               // the lane's piece of a row in even loads; in odd ones, eight rows on, the halves have changed places
        int whole_stages;        // stages whose pieces are all there
        int pieces;
        unsigned past_half_scale;   // what a lane steps back by when the last stage is half of one
        const char* base;
        const char* scale_base;
    };
    __device__ __forceinline__ void start(Loader& l, const Operand& a, const Operand& b, int row0, int col0) const {
        const bool first = wave < 2;  // two wavefronts load A's rows, two B's
        const char* data = first ? a.data : b.data;
        const int64_t stride = first ? a.stride : b.stride;
        const int at = first ? row0 : col0, left = (first ? a.rows : b.rows) - at;
        l.turned = first ? KA : KB;
        l.step = l.turned ? kTurnedRows * stride : kStageBytes;
        l.pieces = first ? a.pieces : b.pieces;
        l.whole_stages = l.pieces ? l.pieces / 8 : INT32_MAX;
        l.line = (unsigned)stride;
        l.depth = first ? a.depth : b.depth;
        l.part_stride = first ? a.part_stride : b.part_stride;
        l.order = first ? a.order : b.order;
        if ((KA || KB) && l.turned) {
            l.base = uniform(data + at * kElement);
#pragma unroll
            for (int i = 0; i < kRowLoads; ++i) {
                const int k = turned_row(i), byte = turned_byte(i) % kTurnedRow;
                const int chunk = turned_piece(byte / (16 * kElement), k) * kElement + (byte >> 4) % kElement, last = left * kElement / 16 - 1;    // of 16 bytes
                l.row[i] = (unsigned)(k * stride) + (chunk < last ? chunk : last) * 16;
            }
            return;
        }
        l.base = uniform(data + at * stride);
        l.piece = (lane & 7) ^ place_of(lane >> 3);
#pragma unroll
        for (int i = 0; i < kRowLoads; ++i) {
            const int row = i * 8 + (lane >> 3), piece = (lane & 7) ^ place_of(row);   // the other wavefronts' rows are multiples of 16 away
            int r = (wave & 1) * (kRowLoads * 8) + row;
            r = r < left ? r : left - 1;
            l.row[i] = (unsigned)(r * stride) + piece * 16;
        }
        if constexpr (Product::kScaled) {
            const int64_t scale_stride = first ? a.scale_stride : b.scale_stride;
            l.scale_base = uniform((const char*)(first ? a.scales : b.scales) + at * scale_stride);
            l.past_half_scale = lane & 1 ? 4 : 0;
#pragma unroll
            for (int i = 0; i < kScaleLoads; ++i) {
                int r = (wave & 1) * (kScaleLoads * 32) + i * 32 + (lane >> 1);
                r = r < left ? r : left - 1;
                l.scale[i] = (unsigned)(r * scale_stride) + (lane & 1) * 4;
            }
        }
    }
    // Turned operands: which byte of the wavefront's operand in a stage the lane's part of load i is, and in which row that is.
    __device__ __forceinline__ int turned_byte(int i) const { return (wave & 1) * (kRowLoads * 1024) + i * 1024 + lane * 16; }
    __device__ __forceinline__ int turned_row(int i) const { return turned_byte(i) / kTurnedRow; }

    // The i-th load of a stage.  LAST: it may be the last one of the contraction, where rows end; half: in the middle of the stage, its second half repeats the first.
    template <bool LAST> __device__ __forceinline__ void load(const Loader& l, int i, int stage, bool half) const {
        const unsigned buffer = smem_address + buffer_of(stage);
        const char* base = l.base;
        stage += first_stage;
        if constexpr (Product::kParts) {
            int segment = 0;
#pragma unroll
            for (int k = 1; k < kSegments; ++k) segment += stage >= k * segment_stages ? 1 : 0;
            stage -= segment * segment_stages;
            base += (int64_t)(l.order >> 2 * segment & 3) * l.part_stride;
        }
        if (i < kRowLoads) {
            unsigned at = l.row[i];
            if constexpr (LAST || Product::kParts) {    // a segment's end may be anywhere
                if ((KA || KB) && l.turned) {
                    const int last = l.depth - 1 - stage * kTurnedRows, k = turned_row(i);    // rows of the stage
                    at -= k > last ? (unsigned)(k - last) * l.line : 0u;
                } else if (half || stage >= l.whole_stages) {    // pieces behind the last one there is, or behind the half, repeat the last before
                    const int piece = i & 1 ? l.piece ^ 4 : l.piece, left = l.pieces ? l.pieces - stage * 8 : 8;
                    const int last = (half && left > 4 ? 4 : left) - 1;
                    at -= piece > last ? (unsigned)(piece - last) * 16 : 0u;
                }
            }
            load_to_lds16(buffer + (wave * kRowLoads + i) * 1024, at, base + stage * l.step);
        } else if constexpr (Product::kScaled) {
            const int k = i - kRowLoads;
            load_to_lds4(buffer + kScaleOffset + (wave * kScaleLoads + k) * 256, l.scale[k] - (LAST && half ? l.past_half_scale : 0),
                         l.scale_base + (int64_t)stage * (kStageBytes / 16));
        }
    }

    __device__ __forceinline__ static i16x4 transposed(const char* p) {
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)p);
    }

    // What a wavefront multiplies in one phase; of a scaled product also its scales, as read and as the instructions take them.
    struct Operands { Frag a[kFrags], b[kFrags]; };
    struct Scales { int a[Product::kScaled ? kFrags : 1], b[Product::kScaled ? kFrags : 1]; };

    // Operand piece f of the wavefront (0..kFrags-1: B's, then A's) for phase `half` of a stage.  Each of the four groups of 16
    // lanes takes a 16-byte piece of eight (which ones in which phase: see the layout above; any order gives the same sum).
    // short_stage: the stage has four pieces, phase 0 takes them.
    __device__ __forceinline__ void read(Operands& to, int f, int stage, int half, bool short_stage) const {
        const bool is_b = f < kFrags;
        const int i = is_b ? f : f - kFrags, group = lane >> 4;
        if ((KA && !is_b) || (KB && is_b)) {
            const int piece = (is_b ? wave & 1 : wave >> 1) * kFrags + i;
            const char* from = smem + buffer_of(stage) + (is_b ? kTile * kStageBytes : 0);
            Frag all;
            if constexpr (kElement == 4) {
                const int k = half * 16 + group * 4;
                const float* p = reinterpret_cast<const float*>(from + k * kTurnedRow + turned_place(piece, k) * 64) + (lane & 15);
#pragma unroll
                for (int e = 0; e < 4; ++e) all[e] = p[e * (kTurnedRow / 4)];
            } else {
                const int k = half * 32 + group * 8 + (lane >> 2 & 3);
                from += k * kTurnedRow + turned_place(piece, k) * 32 + (lane & 3) * 8;    // rows k and k + 4 are shifted alike
                all = __builtin_bit_cast(Frag, __builtin_shufflevector(transposed(from), transposed(from + 4 * kTurnedRow), 0, 1, 2, 3, 4, 5, 6, 7));
            }
            (is_b ? to.b[i] : to.a[i]) = all;
            return;
        }
        const int row = (is_b ? kTile + (wave & 1) * WT : (wave >> 1) * WT) + i * 16 + (lane & 15);
        const int piece = short_stage ? group : Product::kScaled ? 2 * group + half : group + 4 * half;
        (is_b ? to.b[i] : to.a[i]) = *reinterpret_cast<const Frag*>(smem + buffer_of(stage) + row * kStageBytes + ((piece ^ place_of(row)) * 16));
    }
    // The four scale bytes among which the lane's two are.
    __device__ __forceinline__ void read_scales(Scales& to, int f, int stage, bool short_stage) const {
        const bool is_b = f < kFrags;
        const int i = is_b ? f : f - kFrags, group = lane >> 4;
        const int row = (is_b ? kTile + (wave & 1) * WT : (wave >> 1) * WT) + i * 16 + (lane & 15);
        (is_b ? to.b[i] : to.a[i]) = *reinterpret_cast<const int*>(smem + buffer_of(stage) + kScaleOffset + row * 8 + (short_stage ? 0 : (group >> 1) * 4));
    }
    __device__ __forceinline__ void settle(Scales& now, const Scales& raw, bool short_stage) const {
        if constexpr (Product::kScaled) {
            const int group = lane >> 4, shift = short_stage ? group * 8 : (group & 1) * 16;
#pragma unroll
            for (int i = 0; i < kFrags; ++i) {
                now.a[i] = (int)((u32)raw.a[i] >> shift);
                now.b[i] = (int)((u32)raw.b[i] >> shift);
            }
        }
    }

    // Phase HALF of a stage: multiplies `now` while reading the operands of the next phase and, where LOAD says so, issuing a stage's loads:
    // at most one of each between two matrix instructions, fenced so that they stay there (in clumps they hold the wavefront
    // up: 5 % of the rate at 4096 x 4096 x 8192).  The reads end a quarter before the phase does, so the next finds its operands.
    enum { kNoLoad = 0, kLoad = 1, kLoadLast = 2 };
    template <int HALF, int LOAD>
    __device__ __forceinline__ void phase(const Operands& now, const Scales& scales, Operands& next, Scales& next_scales, int read_stage,
                                          bool read_short, const Loader& l, int load_stage, bool load_half) {
        constexpr int kAll = kFrags * kFrags;
        constexpr int kScaleReads = Product::kScaled && HALF == 1 ? kFrags : 0;   // two at a time
        constexpr int kReads = 2 * kFrags + kScaleReads;
        constexpr int kReadWithin = kAll >= 16 ? kAll - kAll / 4 : kAll;
#pragma unroll
        for (int q = 0; q < kAll; ++q) {
            if constexpr (LOAD != kNoLoad) {
#pragma unroll
                for (int k = q * kLoads / kAll; k < (q + 1) * kLoads / kAll; ++k) {
                    load<LOAD == kLoadLast>(l, k, load_stage, load_half);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int k = q * kReads / kReadWithin; k < (q + 1) * kReads / kReadWithin && k < kReads; ++k) {
                if (k < kScaleReads) {
                    read_scales(next_scales, 2 * k, read_stage, read_short);
                    read_scales(next_scales, 2 * k + 1, read_stage, read_short);
                } else {
                    read(next, k - kScaleReads, read_stage, 1 - HALF, read_short);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            constexpr int kOnly = Product::kScaled ? 1 : 0;
            Product::template multiply<HALF>(now.a[q / kFrags], now.b[q % kFrags], acc[q / kFrags][q % kFrags], scales.a[q / kFrags * kOnly], scales.b[q % kFrags * kOnly]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // Says that an accumulator lives in accumulator registers here.
    __device__ __forceinline__ static void keep(f32x4& c) { asm volatile("" : "+a"(c)); }

    // Waits for LDS reads and for all loads but those of the last `later` stages (of kStages at most).
    __device__ __forceinline__ static void wait_behind(int later) {
        if constexpr (kStages > 3) {
            if (later >= 3) { wait_loads_and_lds<3 * kLoads>(); return; }
        }
        if constexpr (kStages > 2) {
            if (later >= 2) { wait_loads_and_lds<2 * kLoads>(); return; }
        }
        if (later >= 1) wait_loads_and_lds<kLoads>();
        else wait_loads_and_lds<0>();
    }

    // The matrix instructions' last results are written.
    __device__ __forceinline__ static void settled() { asm volatile("s_nop 15\n\ts_nop 3" : : : "memory"); }

    // total += acc, acc = 0.  Every stage before is multiplied.
    __device__ __forceinline__ void flush() {
        settled();
#pragma unroll
        for (int i = 0; i < kFrags; ++i)
#pragma unroll
            for (int j = 0; j < kFrags; ++j) {
                keep(acc[i][j]);
                total[i][j] += acc[i][j];
                acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                keep(acc[i][j]);
            }
    }

    // acc = the product's tile at (row0, col0) over rows of `row_bytes` > 0.
    __device__ __forceinline__ void multiply(const Operand& a, const Operand& b, int row0, int col0, int row_bytes) {
#pragma unroll
        for (int i = 0; i < kFrags; ++i)
#pragma unroll
            for (int j = 0; j < kFrags; ++j) {
                acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                keep(acc[i][j]);
                if constexpr (kTwoSums) total[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        const int stages = (row_bytes + kStageBytes - 1) / kStageBytes;
        const bool odd = (row_bytes / kHalfBytes) & 1;   // the last stage is a short one
        Loader l;
        start(l, a, b, row0, col0);
#pragma unroll
        for (int stage = 0; stage < kStages; ++stage) {
            if (stage >= stages) break;
#pragma unroll
            for (int k = 0; k < kLoads; ++k) load<true>(l, k, stage, odd && stages == stage + 1);
        }
        wait_behind(stages - 1);
        meet();
        Operands even, uneven;
        Scales raw, scales;
        const bool first_short = odd && stages == 1;
#pragma unroll
        for (int f = 0; f < 2 * kFrags; ++f) {
            read(even, f, 0, 0, first_short);
            if constexpr (Product::kScaled) read_scales(raw, f, 0, first_short);
        }
        int s = 0;
        for (; s + kStages + 1 < stages; ++s) {
            settle(scales, raw, false);
            phase<0, kNoLoad>(even, scales, uneven, raw, s, false, l, 0, false);
            wait_loads_and_lds<(kStages - 2) * kLoads>();  // stage s is in registers, stage s + 1 in LDS
            meet();
            phase<1, kLoad>(uneven, scales, even, raw, s + 1, false, l, s + kStages, false);
            if constexpr (kTwoSums) {
                if (s % kFlushStages == kFlushStages - 1) flush();
            }
        }
        if (s + kStages < stages) {   // the same with the loads of the last stage
            settle(scales, raw, false);
            phase<0, kNoLoad>(even, scales, uneven, raw, s, false, l, 0, false);
            wait_loads_and_lds<(kStages - 2) * kLoads>();
            meet();
            phase<1, kLoadLast>(uneven, scales, even, raw, s + 1, odd && s + 2 == stages, l, s + kStages, odd);
            ++s;
        }
        for (;; ++s) {
            const bool last = s + 1 == stages;
            settle(scales, raw, odd && last);
            phase<0, kNoLoad>(even, scales, uneven, raw, s, false, l, 0, false);
            wait_behind(stages - s - 2);
            meet();
            if (last && odd) break;
            phase<1, kNoLoad>(uneven, scales, even, raw, s + 1, odd && s + 2 == stages, l, 0, false);
            if (last) break;
        }
        settled();
#pragma unroll
        for (int i = 0; i < kFrags; ++i)
#pragma unroll
            for (int j = 0; j < kFrags; ++j) {
                keep(acc[i][j]);
                if constexpr (kTwoSums) {
                    acc[i][j] += total[i][j];
                    keep(acc[i][j]);
                }
            }
        meet();  // the epilogue writes over the buffers
    }

    // ------------------------------------------------------------------------------------------- epilogue
    // Hands the tile to `out` row by row: out.row(i, j, in, v) gets v[0..7] = C[i][j .. j+7] (i, j counted in the whole result, j
    // a multiple of 8 and the same for all rows that a lane gets, said before by out.begin(j)) and, with out.kColumns,
    // leaves in v what out.column(i, j, w) then gets column by column: w[0..7] = rows i .. i+7 of column j.  Consecutive lanes get
    // consecutive pieces of a row (of eight rows of a column).  What out reads from memory for a row it reads in
    // out.load(i, j, in), called a strip ahead.
    template <class Out> __device__ __forceinline__ void finish(int row0, int col0, Out& out) {
        float* strip = reinterpret_cast<float*>(smem + wave * kStripBytes);
        constexpr int kPieces = WT / 8;              // 8-value pieces of a row
        constexpr int kRowsAtOnce = 64 / kPieces;    // WT = 96: five rows, four lanes sit out
        constexpr int kPasses = (32 + kRowsAtOnce - 1) / kRowsAtOnce;
        constexpr int kStrips = WT / 32;
        const int r0 = row0 + (wave >> 1) * WT, c0 = col0 + (wave & 1) * WT;
        const int first = lane / kPieces, piece = lane % kPieces * 8;
        const bool idle = first >= kRowsAtOnce;
        typename Out::In in[kPasses];
        out.begin(c0 + piece);
#pragma unroll
        for (int k = 0; k < kPasses; ++k)
            if (!idle && first + k * kRowsAtOnce < 32) out.load(r0 + first + k * kRowsAtOnce, c0 + piece, in[k]);
#pragma unroll 1
        for (int s = 0; s < kStrips; ++s) {
            // the accumulators are named registers: one copy of this part for each strip, one of the rest
            if (s == 0) lay_out<0>(strip);
            else if (s == 1) lay_out<1>(strip);
            else if (s == 2) lay_out<2>(strip);
            else lay_out<3>(strip);
            same_wave();
#pragma unroll
            for (int k = 0; k < kPasses; ++k) {
                const int r = first + k * kRowsAtOnce;
                if (idle || r >= 32) continue;
                f32x4* p = reinterpret_cast<f32x4*>(strip + r * kStripStride + piece);
                const f32x4 lo = p[0], hi = p[1];
                float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                const typename Out::In now = in[k];
                if (s + 1 < kStrips) out.load(r0 + (s + 1) * 32 + r, c0 + piece, in[k]);
                out.row(r0 + s * 32 + r, c0 + piece, now, v);
                if constexpr (Out::kColumns) {
                    p[0] = f32x4{v[0], v[1], v[2], v[3]};
                    p[1] = f32x4{v[4], v[5], v[6], v[7]};
                }
            }
            if constexpr (Out::kColumns) {
                same_wave();
                if (out.columns()) {
                    for (int k = lane; k < WT * 4; k += 64) {
                        const int col = k >> 2, rows = (k & 3) * 8;
                        float w[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) w[e] = strip[(rows + e) * kStripStride + col];
                        out.column(r0 + s * 32 + rows, c0 + col, w);
                    }
                }
            }
            same_wave();
        }
    }
    template <int S> __device__ __forceinline__ void lay_out(float* strip) const {
        if constexpr (S < WT / 32) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < kFrags; ++j)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        strip[(h * 16 + (lane >> 4) * 4 + k) * kStripStride + j * 16 + (lane & 15)] = acc[2 * S + h][j][k];
        }
    }
    // A wavefront's LDS accesses take effect in order; this keeps the compiler from reordering them.
    __device__ __forceinline__ static void same_wave() {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
};

// ------------------------------------------------------------------------------------------- which tile a workgroup takes
// Workgroup b runs on accelerator die b % 8, each with an L2 of its own: every die takes a contiguous run of the tiles.
// `seat` is the workgroup's place among its die's; a grid has 8 * seats_of(tiles) workgroups, up to seven of them without a
// tile (negative).
__host__ __device__ __forceinline__ int64_t seats_of(int64_t tiles) { return (tiles + 7) >> 3; }
__device__ __forceinline__ int64_t tile_of_seat(int die, int64_t seat, int64_t tiles) {
    const int64_t per = tiles >> 3, rest = tiles & 7;
    if (seat >= per + (die < rest ? 1 : 0)) return -1;
    return die * per + (die < rest ? die : rest) + seat;
}
// Tile t of a result of `rows` x `cols` tiles, in bands of four rows, column by column: 32 consecutive tiles (a die's
// compute units) share twelve operand panels.
__device__ __forceinline__ void tile_at(int t, int rows, int cols, int& i, int& j) {
    const int band = t / (4 * cols), left = t - band * 4 * cols;
    const int height = rows - band * 4 < 4 ? rows - band * 4 : 4;
    i = band * 4 + left % height;
    j = left / height;
}
// The same for the tiles on and above the diagonal of a symmetric result of n x n tiles: n (n + 1) / 2 of them.
__device__ __forceinline__ void tile_at_symmetric(int t, int n, int& i, int& j) {
    int first = 0;
    for (;;) {
        const int height = n - first < 4 ? n - first : 4;
        const int corner = height * (height + 1) / 2, in_band = corner + (n - first - height) * height;
        if (t < in_band) {
            if (t < corner) {
                int k = 0;
                while (t >= k + 1) t -= ++k;   // column k of the corner has k + 1 tiles
                i = first + t;
                j = first + k;
            } else {
                t -= corner;
                i = first + t % height;
                j = first + height + t / height;
            }
            return;
        }
        t -= in_band;
        first += 4;
    }
}

// ------------------------------------------------------------------------------------------- which tile a launch uses
// Measured times of tiles, in us: a workgroup alone on its compute unit, and with the unit full of them; `each` per value
// contracted.
struct TileCost { int wt, stages, resident; double start, each, start_full, each_full; };

// What `tiles` of them take on `cus` compute units, `length` values contracted: full rounds, then what is left.
inline double tiles_time(const TileCost& c, double tiles, double length, int cus) {
    const double seats = (double)cus * c.resident, rounds = __builtin_floor(tiles / seats);
    const double full = c.start_full + c.each_full * length, alone = c.start + c.each * length;
    const double left = __builtin_ceil((tiles - rounds * seats) / cus);   // on the fullest unit
    const double last = left == 0 ? 0.0 : c.resident == 1 ? full : alone + (full - alone) * (left - 1) / (c.resident - 1);
    return rounds * full + last;
}

// A result of rows x cols in two launches: its first `lines` tile rows (columns) in one kind of tile, which fill whole rounds, what is left in
// another, two or more on a compute unit.  One kind alone (rest.wt = 0) where that takes no longer.  4096 x 14336 over 4096 values
// is three and a half rounds of 256 x 256 tiles: with the last half
// in one round of 128 x 128 tiles the iteration takes 3.48 ms, in one launch 3.61; a scaled product's 145 us become 141.
struct Cut { TileCost tile, rest; bool columns; int lines; double time; };
constexpr double kLaunchTime = 6.0;   // us that a second launch costs

inline int64_t tiles_of(int64_t rows, int64_t cols, int wt) { return ((rows + 2 * wt - 1) / (2 * wt)) * ((cols + 2 * wt - 1) / (2 * wt)); }

// `before` tiles over before_length values(wt) are in the launch already, ahead of this result.
template <int N, class F> Cut best_cut(const TileCost (&costs)[N], int64_t rows, int64_t cols, double length, F before, double before_length, int cus) {
    Cut best{};
    for (const TileCost& c : costs) {
        const double ahead = before(c.wt);
        const auto time = [&](double tiles) { return tiles_time(c, ahead + tiles, (ahead * before_length + tiles * length) / (ahead + tiles), cus); };
        const int64_t across[2] = {(cols + 2 * c.wt - 1) / (2 * c.wt), (rows + 2 * c.wt - 1) / (2 * c.wt)};   // tiles in a row, in a column
        const double whole = time((double)(across[0] * across[1]));
        if (!best.tile.wt || whole < best.time) best = Cut{c, TileCost{}, false, 0, whole};
        const double seats = (double)cus * c.resident, full = __builtin_floor((ahead + (double)(across[0] * across[1])) / seats) * seats - ahead;
        for (int columns = 0; columns < 2; ++columns) {
            const int64_t lines = (int64_t)(full / (double)across[columns]);
            if (full <= 0.0 || lines <= 0 || lines >= across[1 - columns]) continue;
            const double first = time((double)(lines * across[columns])) + kLaunchTime;
            const int64_t left_rows = columns ? rows : rows - lines * 2 * c.wt, left_cols = columns ? cols - lines * 2 * c.wt : cols;
            for (const TileCost& r : costs) {
                const double both = first + tiles_time(r, (double)tiles_of(left_rows, left_cols, r.wt), length, cus);
                if (both < best.time) best = Cut{c, r, columns != 0, (int)lines, both};
            }
        }
    }
    return best;
}

}  // namespace fo
