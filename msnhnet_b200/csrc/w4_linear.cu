// Products with 4-bit weights (msnh_b200_w4_pack, msnh_b200_w4_linear).
//
// y = x_scale * sum over groups of scale * sum_k x (code - zero), + bias. The packed weights are read once; with few rows their bytes bound
// it, and right behind them the instructions that make operands of codes, with 64 rows the products. Three kernels, chosen at the end of
// this file by rows, tiles and k with what either side measured. One fp16 token times 8192 x 28672 (122 MB): 28.4 us, 4.3 TB/s; times
// 4096 x 4096 5.9 us; seven 8-bit rows times 5120 x 13824 19 us (2.05 TB/s); 64 fp16 rows times 8192 x 8192 43.5 us.
#include <cooperative_groups.h>
#include "token_ops.h"
#include "token_types.cuh"

namespace msnh {
namespace {

// Packed weights: units of 16 rows by 128 values, the units of a 16-row tile one behind the other. A unit is 1024 bytes of codes, then
// for each of its 1, 2 or 4 spans (128, 64 or 32 values: the most that always lie in one group) eight records of the scales (fp16 or
// fp32) and zero points (a byte each) of rows r and r + 8, 8 or 16 bytes. Codes beyond n and k are 0.
// Of the codes, 16 bytes of each half (64 values, 512 bytes) belong to a lane of the warp that reads it: lane l has rows l / 4 and
// l / 4 + 8, and in its words 2 s and 2 s + 1 (one for either row) the eight values from 32 * s + 8 * (l % 4) on: byte i has value i in its
// low and value 4 + i in its high half. Two masks make 8-bit A operands of m16n8k32 of a word, four make 16-bit ones of m16n8k16, with k in
// an order that the B operand follows, so nothing is moved between lanes.
constexpr int kTileRows = 16, kUnitK = 128, kCodeBytes = 1024;

struct W4Layout {
    int n, k, group, tiles, units, groups, wide, spans;          // units: of a tile; wide: scales in fp32; spans: of a unit
    size_t unit_bytes, bytes;
    W4Layout(const MsnhB200W4 &w)
        : n(w.n), k(w.k), group(w.group), tiles((w.n + kTileRows - 1) / kTileRows), units((w.k + kUnitK - 1) / kUnitK),
          groups((w.k + w.group - 1) / w.group), wide(w.scale_dtype != MSNH_B200_F16), spans(w.group % 128 == 0 ? 1 : w.group % 64 == 0 ? 2 : 4) {
        unit_bytes = kCodeBytes + static_cast<size_t>(spans) * 8 * (wide ? 16 : 8);
        bytes = static_cast<size_t>(tiles) * units * unit_bytes;
    }
};

template <typename S> struct Record { S scale[2]; uint8_t zero[2], rest[sizeof(S) * 2 - 2]; };

__device__ __forceinline__ int code_at(const uint8_t *codes, long long stride, int n, int k, int row, int at) {
    if (row >= n || at >= k) return 0;
    return codes[row * stride + at / 2] >> (at % 2 * 4) & 15;
}

__global__ void w4_pack_codes_kernel(const uint8_t *codes, long long stride, int n, int k, int units, size_t unit_bytes, long long words, uint8_t *out) {
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < words; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int in_unit = static_cast<int>(i % 256), half = in_unit / 128, lane = in_unit / 4 % 32, word_of = in_unit % 4;
        const long long unit = i / 256;
        const int row = static_cast<int>(unit / units) * kTileRows + lane / 4 + word_of % 2 * 8;
        const int at = static_cast<int>(unit % units) * kUnitK + 64 * half + 32 * (word_of / 2) + 8 * (lane % 4);
        uint32_t word = 0;
#pragma unroll
        for (int v = 0; v < 8; ++v) word |= static_cast<uint32_t>(code_at(codes, stride, n, k, row, at + v)) << (v % 4 * 8 + v / 4 * 4);
        *reinterpret_cast<uint32_t *>(out + unit * unit_bytes + in_unit * 4) = word;
    }
}

template <typename S, typename Out>
__global__ void w4_pack_records_kernel(const S *scales, const uint8_t *zeros, int n, int k, int units, int spans, int group, int groups, size_t unit_bytes,
                                       long long count, uint8_t *out) {
    for (long long i = blockIdx.x * static_cast<long long>(blockDim.x) + threadIdx.x; i < count; i += static_cast<long long>(gridDim.x) * blockDim.x) {
        const int pair = static_cast<int>(i % 8), span = static_cast<int>(i / 8 % spans);
        const long long unit = i / 8 / spans, at = unit % units * kUnitK + span * (kUnitK / spans);
        const long long g = at / group;
        Record<Out> r = {};
        for (int half = 0; half < 2; ++half) {
            const long long row = unit / units * kTileRows + pair + 8 * half;
            const bool there = row < n && at < k;
            r.scale[half] = there ? static_cast<Out>(to_float(scales[row * groups + g])) : static_cast<Out>(0.f);
            r.zero[half] = there && zeros ? zeros[row * groups + g] & 15 : 8;
        }
        reinterpret_cast<Record<Out> *>(out + unit * unit_bytes + kCodeBytes)[span * 8 + pair] = r;
    }
}

struct W4Params {
    const uint8_t *packed;
    const void *x;
    void *y;
    const float *x_scale, *bias;
    long long x_stride, y_stride;
    long long unit_bytes;
    int n, k, tiles, units, rows;
    int dtype, wide, spans, vectors, out_dtype;
    int split, share, block_units;           // warps that share a tile's k in a block; units of k of each, of the block at most
    int ring_at, x_at, meta_at;              // of the rings and the activations, in shared memory
    uint8_t *digits_made, *meta_made;        // digits (or 16-bit operands) and what belongs to them in the workspace, or null
    int *error;                              // where the host learns of a wait that ran out
    uint32_t exponents;                      // of the operands' type (a parameter, so that the compiler takes it for a variable)
};

constexpr int kWarps = 16, kSummers = 4, kThreads = (kWarps + kSummers) * 32;      // warps that multiply, and that add up
constexpr int kMostRanks = 8;                // blocks of a cluster

__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// The A operand's element type for activations of type X, and how many operands of that type an activation becomes: fp16, bf16 and 8-bit
// values are operands themselves, an fp32 value is the sum of three bf16 ones (8 bits of it each), whose products with a code are exact.
template <typename X> struct Operand { using Type = X; static constexpr int kParts = 1; };
template <> struct Operand<__nv_fp8_e4m3> { using Type = __half; static constexpr int kParts = 1; };
template <> struct Operand<float> { using Type = __nv_bfloat16; static constexpr int kParts = 3; };

template <typename H> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    H v[2] = {from_float<H>(a), from_float<H>(b)};
    uint32_t r;
    memcpy(&r, v, 4);
    return r;
}
// the three bf16 parts of two fp32 values
__device__ __forceinline__ void split2(float a, float b, uint32_t &high, uint32_t &middle, uint32_t &low) {
    // (the largest fp32 values would be rounded to an infinity: their first part is the largest bf16 value)
    constexpr float kMost = 3.3895313892515355e38f;
    const bool fa = fabsf(a) <= 3.4028235e38f, fb = fabsf(b) <= 3.4028235e38f;
    high = pack2<__nv_bfloat16>(fa ? fminf(fmaxf(a, -kMost), kMost) : a, fb ? fminf(fmaxf(b, -kMost), kMost) : b);
    // (what is left of an infinity or NaN is 0: the first part carries it)
    const float ra = fa ? a - __uint_as_float(high << 16) : 0.f, rb = fb ? b - __uint_as_float(high & 0xffff0000u) : 0.f;
    middle = pack2<__nv_bfloat16>(ra, rb);
    low = pack2<__nv_bfloat16>(ra - __uint_as_float(middle << 16), rb - __uint_as_float(middle & 0xffff0000u));
}

// pairs 01 23 45 67 to 02 13 46 57
__device__ __forceinline__ void interleave(uint32_t (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t a = v[i], b = v[i + 1];
        v[i] = __byte_perm(a, b, 0x5410);
        v[i + 1] = __byte_perm(a, b, 0x7632);
    }
}

// Eight values of a row: read whole (aligned, all there), or the first `left` of them and zeros; then as operands, two k-steps of two
// registers a part, values 0 and 2, 1 and 3, 4 and 6, 5 and 7.
template <typename X> struct Raw {
    uint4 v;
    __device__ __forceinline__ void load(const X *row) { v = __ldg(reinterpret_cast<const uint4 *>(row)); }
    __device__ __forceinline__ void load(const X *row, int left) {
        X one[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) one[i] = i < left ? row[i] : from_float<X>(0.f);
        memcpy(&v, one, 16);
    }
    __device__ __forceinline__ void operands(uint32_t (&out)[1][4]) const {
        out[0][0] = v.x; out[0][1] = v.y; out[0][2] = v.z; out[0][3] = v.w;
        interleave(out[0]);
    }
};
template <> struct Raw<float> {
    float v[8];
    __device__ __forceinline__ void load(const float *row) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(row)), b = __ldg(reinterpret_cast<const float4 *>(row) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    __device__ __forceinline__ void load(const float *row, int left) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? row[i] : 0.f;
    }
    __device__ __forceinline__ void operands(uint32_t (&out)[3][4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) split2(v[i / 2 * 4 + i % 2], v[i / 2 * 4 + i % 2 + 2], out[0][i], out[1][i], out[2][i]);
    }
};
template <> struct Raw<__nv_fp8_e4m3> {
    uint2 v;
    __device__ __forceinline__ void load(const __nv_fp8_e4m3 *row) { v = __ldg(reinterpret_cast<const uint2 *>(row)); }
    __device__ __forceinline__ void load(const __nv_fp8_e4m3 *row, int left) {
        uint8_t bytes[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) bytes[i] = i < left ? reinterpret_cast<const uint8_t *>(row)[i] : 0;
        memcpy(&v, bytes, 8);
    }
    __device__ __forceinline__ void operands(uint32_t (&out)[1][4]) const {
        uint16_t pairs[4];
        memcpy(pairs, &v, 8);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(pairs[i], __NV_E4M3);
            memcpy(&out[0][i], &h, 4);
        }
        interleave(out[0]);
    }
};

// (w & mask) | exponents in one instruction, which takes one constant at most: the exponents come in a register
template <uint32_t kMask> __device__ __forceinline__ uint32_t masked_or(uint32_t w, uint32_t exponents) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "n"(kMask), "r"(exponents));
    return r;
}
// The 16-bit operands of a word of codes, less their row's zero point: values 0 and 2, 1 and 3, 4 and 6, 5 and 7. fp16: a half-byte below
// the exponent of 1024 is 1024 + code, one four bits higher 1024 + 16 code; bf16 has seven bits behind its leading one, so every half-byte
// is moved to the lowest place: 128 + code. All exact. Operands are 1 / kUnit of the codes: bf16 and fp32 activations go up to 2^128, and the
// sum of a span, up to 15 * 128 of them, must not be infinite where its scale would bring it back.
template <typename H> struct Zero;
template <> struct Zero<__half> {
    static constexpr float kUnit = 1.f;
    static constexpr uint32_t kExponents = 0x64006400u;
    __half2 low, high;
    __device__ __forceinline__ void set(uint32_t z) {
        const uint32_t a = (0xe400u + z) * 0x10001u, b = (0xd400u + 16 * z) * 0x10001u;        // -(1024 + zero), -(64 + zero)
        memcpy(&low, &a, 4);
        memcpy(&high, &b, 4);
    }
    __device__ __forceinline__ void operand(uint32_t w, uint32_t exponents, uint32_t (&out)[4]) const {
        const __half2 sixteenth = __half2half2(__float2half_rn(0.0625f));
        const uint32_t above = w >> 8;
        const uint32_t raw[4] = {masked_or<0x000f000fu>(w, exponents), masked_or<0x000f000fu>(above, exponents), masked_or<0x00f000f0u>(w, exponents),
                                 masked_or<0x00f000f0u>(above, exponents)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __half2 v;
            memcpy(&v, &raw[i], 4);
            v = i / 2 ? __hfma2(v, sixteenth, high) : __hadd2(v, low);
            memcpy(&out[i], &v, 4);
        }
    }
};
template <> struct Zero<__nv_bfloat16> {
    static constexpr float kUnit = 2048.f;
    static constexpr uint32_t kExponents = 0x3d803d80u;
    __nv_bfloat162 low;
    __device__ __forceinline__ void set(uint32_t z) {
        const uint32_t a = (0xbd80u + z) * 0x10001u;                                           // -(128 + zero) / kUnit
        memcpy(&low, &a, 4);
    }
    __device__ __forceinline__ void operand(uint32_t w, uint32_t exponents, uint32_t (&out)[4]) const {
        const uint32_t raw[4] = {masked_or<0x000f000fu>(w, exponents), masked_or<0x000f000fu>(w >> 8, exponents), masked_or<0x000f000fu>(w >> 4, exponents),
                                 masked_or<0x000f000fu>(w >> 12, exponents)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __nv_bfloat162 v;
            memcpy(&v, &raw[i], 4);
            v = __hadd2(v, low);
            memcpy(&out[i], &v, 4);
        }
    }
};

// Scales and zero points of a lane's two rows, from a record in shared memory.
__device__ __forceinline__ void take_record(uint32_t record, int wide, float2 &scale, uint32_t &z0, uint32_t &z8) {
    uint32_t zeros;
    if (wide) {
        asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(scale.x), "=f"(scale.y) : "r"(record) : "memory");
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(zeros) : "r"(record + 8) : "memory");
    } else {
        uint32_t both;
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(both), "=r"(zeros) : "r"(record) : "memory");
        __half2 pair;
        memcpy(&pair, &both, 4);
        scale = __half22float2(pair);
    }
    z0 = zeros & 255;
    z8 = zeros >> 8 & 255;
}
__device__ __forceinline__ uint4 load_shared(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

template <typename H> __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<H, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void store(const W4Params &p, int m, int row, float v) {
    const float y = v * (p.x_scale ? p.x_scale[m] : 1.f) + (p.bias ? p.bias[row] : 0.f);
    const long long at = m * p.y_stride + row;
    if (p.out_dtype == MSNH_B200_F32) static_cast<float *>(p.y)[at] = y;
    else if (p.out_dtype == MSNH_B200_F16) static_cast<__half *>(p.y)[at] = __float2half_rn(y);
    else static_cast<__nv_bfloat16 *>(p.y)[at] = __float2bfloat16_rn(y);
}

// A block stays for its share of the tiles, kTiles at a time for each of its sets of `split` warps; the warps of a set share the tiles' k,
// and so may the blocks of a cluster. What both kernels need of that.
template <int kTiles> struct Share {
    int lane, warp, ranks, rank, sets, turn, from, to, mine;     // turn: tiles of one; this block's, and this warp's first one
    int begin, first, count;                                     // units of k: the block's first, the warp's first, how many
    int block_units;
    __device__ __forceinline__ Share(const W4Params &p, int cluster_blocks, int cluster_rank) {
        lane = threadIdx.x % 32;
        warp = threadIdx.x / 32;
        ranks = cluster_blocks;
        rank = cluster_rank;
        sets = kWarps / p.split;
        turn = kTiles * sets;
        const int place = blockIdx.x / ranks, places = gridDim.x / ranks;
        from = static_cast<int>(static_cast<long long>(p.tiles) * place / places);
        to = static_cast<int>(static_cast<long long>(p.tiles) * (place + 1) / places);
        mine = from + warp / p.split * kTiles;
        begin = min(rank * p.split * p.share, p.units);
        block_units = min(begin + p.split * p.share, p.units) - begin;
        first = min(begin + warp % p.split * p.share, p.units);
        count = warp < kWarps ? min(first + p.share, p.units) - first : 0;
    }
};

// A warp's units of every turn's tiles, one turn after the other, through a ring with cp.async. Of a tile that is not the block's nothing is
// copied, and what its sums are made of is never stored.
template <int kTiles, int kAhead> struct Units {
    const uint8_t *codes;
    long long unit_bytes, tile_bytes, next_turn;
    uint32_t ring, ring_end, fill, slot;
    int pitch, copy_tile, to, turn, copied, count, lane;
    bool copies_record;
    __device__ __forceinline__ Units(const W4Params &p, const Share<kTiles> &s, uint32_t rings) {
        lane = s.lane;
        pitch = static_cast<int>(p.unit_bytes);
        unit_bytes = p.unit_bytes;
        tile_bytes = p.units * p.unit_bytes;
        next_turn = s.turn * tile_bytes - s.count * p.unit_bytes;
        codes = p.packed + s.mine * tile_bytes + s.first * p.unit_bytes + lane * 16;
        copy_tile = s.mine;
        to = s.to;
        turn = s.turn;
        count = s.count;
        copied = 0;
        ring = fill = slot = rings + s.warp * kAhead * kTiles * pitch;
        ring_end = ring + kAhead * kTiles * pitch;
        copies_record = lane * 16 < pitch - kCodeBytes;
        if (count && s.warp < kWarps)
#pragma unroll 1
            for (int u = 0; u < kAhead - 1; ++u) copy();
    }
    __device__ __forceinline__ void copy() {
#pragma unroll
        for (int r = 0; r < kTiles; ++r)
            if (copy_tile + r < to) {
                const uint8_t *at = codes + r * tile_bytes;
                const uint32_t into = fill + r * pitch + lane * 16;
                copy16(into, at);
                copy16(into + 512, at + 512);
                if (copies_record) copy16(into + 1024, at + 1024);
            }
        copy_commit();
        codes += unit_bytes;
        if (++copied == count) {
            copied = 0;
            copy_tile += turn;
            codes += next_turn;
        }
        fill += kTiles * pitch;
        if (fill == ring_end) fill = ring;
    }
    __device__ __forceinline__ void wait() {                     // for the unit at `slot`; the one behind it may be overwritten then
        copy_wait<kAhead - 2>();
        __syncwarp();                                            // (records are other lanes' copies)
        copy();
    }
    __device__ __forceinline__ void next() {
        slot += kTiles * pitch;
        if (slot == ring_end) slot = ring;
    }
};

// The way of a turn's sums [warp][column][row] from the warps that multiply to those that add up: `full` counts the former's arrivals,
// `empty` the latter's. Neither waits for its own kind, so the copies run on meanwhile. The waits have a limit (0.8 s, where the longest
// turn, of k = 2^27, takes 50 ms), after which the host learns of it and the block ends.
constexpr long long kWaitCycles = 1500000000LL;
struct Handover { uint64_t full, empty; };
__device__ __forceinline__ uint32_t shared_address(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void barrier_init(uint64_t *b, int count) { asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(shared_address(b)), "r"(count) : "memory"); }
__device__ __forceinline__ void barrier_arrive(uint64_t *b) { asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(shared_address(b)) : "memory"); }
__device__ __forceinline__ bool barrier_wait(uint64_t *b, int parity, int *error) {
    const auto there = [&] {
        uint32_t done;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(done) : "r"(shared_address(b)), "r"(parity) : "memory");
        return done != 0;
    };
    if (there()) return true;
    for (const long long began = clock64(); clock64() - began <= kWaitCycles;)
        if (there()) return true;
    report_error(error, DEV_ERR_WAIT_SUMS);
    return false;
}

// The outputs of a turn, in a fixed order: four threads an output, each every fourth of the warps that share a tile's k. sums: [warp][row of
// the activations][row of the tiles]. `threads`: a multiple of 32.
template <int kRows, typename Put>
__device__ __forceinline__ void add_up(const W4Params &p, int sets, int columns, const float *sums, int thread, int threads, Put put) {
    const int per_set = kRows * p.rows, each = kRows * columns;
    for (int i = thread; i < sets * per_set * 4; i += threads) {                // (a multiple of 64)
        const int o = i / 4, set = o / per_set, in_set = o - set * per_set;
        const float *from = sums + set * p.split * each + in_set;
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < kWarps / 4; ++j) {
            const int w = j * 4 + i % 4;
            if (w < p.split) v += from[w * each];
        }
        v += __shfl_xor_sync(~0u, v, 1);
        v += __shfl_xor_sync(~0u, v, 2);
        if (i % 4 == 0) put(o, set * (kRows / kTileRows) + in_set % kRows / kTileRows, in_set % kTileRows, in_set / kRows, v);
    }
}

// What a kernel does with a block's turns: multiply(tile) leaves a warp's sums in registers, leave(to) puts them down.
// seen(m, v) is told of every output.
template <int kTiles, int kCount, typename Cluster, typename Multiply, typename Leave, typename Seen>
__device__ __forceinline__ void turns(const W4Params &p, const Share<kTiles> &s, Cluster &cluster, float *sums, Handover &hand, Multiply multiply, Leave leave, Seen seen) {
    constexpr int kRows = kTiles * kTileRows;
    const auto put = [&](int tile, int place, int row, int m, float v) {
        if (tile + place < s.to && (tile + place) * kTileRows + row < p.n) {
            seen(m, v);
            store(p, m, (tile + place) * kTileRows + row, v);
        }
    };
    if (s.ranks > 1) {
        float *const outputs = sums + kWarps * kRows * kCount;
        for (int tile = s.from; tile < s.to; tile += s.turn) {
            if (s.warp < kWarps) {
                multiply();
                leave(sums + s.warp * kRows * kCount);
            }
            __syncthreads();
            add_up<kRows>(p, s.sets, kCount, sums, threadIdx.x, kThreads, [&](int o, int, int, int, float v) { outputs[o] = v; });
            cluster.sync();
            for (int o = s.rank * kThreads + threadIdx.x; o < s.sets * kRows * p.rows; o += s.ranks * kThreads) {
                float v = 0.f, others[kMostRanks];               // (all reads are under way before the first is added)
#pragma unroll
                for (int q = 0; q < kMostRanks; ++q)
                    if (q < s.ranks) others[q] = *cluster.map_shared_rank(&outputs[o], q);
#pragma unroll
                for (int q = 0; q < kMostRanks; ++q)
                    if (q < s.ranks) v += others[q];
                const int set = o / (kRows * p.rows), m = o % (kRows * p.rows) / kRows, row = o % kRows;
                put(tile, set * kTiles + row / kTileRows, row % kTileRows, m, v);
            }
            cluster.sync();                                      // (no block goes on while another reads its sums)
        }
        return;
    }
    if (s.to - s.from <= s.turn) {                               // (one turn: all can add up)
        if (s.warp < kWarps && s.from < s.to) {
            multiply();
            leave(sums + s.warp * kRows * kCount);
        }
        __syncthreads();
        if (s.from < s.to) add_up<kRows>(p, s.sets, kCount, sums, threadIdx.x, kThreads, [&](int, int place, int row, int m, float v) { put(s.from, place, row, m, v); });
        return;
    }
    int parity = 0;
    if (s.warp < kWarps) {
        for (int tile = s.from; tile < s.to; tile += s.turn, parity ^= 1) {
            multiply();
            if (tile != s.from && !barrier_wait(&hand.empty, parity ^ 1, p.error)) return;
            leave(sums + s.warp * kRows * kCount);
            __syncwarp();
            if (s.lane == 0) barrier_arrive(&hand.full);
        }
    } else {
        for (int tile = s.from; tile < s.to; tile += s.turn, parity ^= 1) {
            if (!barrier_wait(&hand.full, parity, p.error)) return;
            add_up<kRows>(p, s.sets, kCount, sums, threadIdx.x - kWarps * 32, kSummers * 32, [&](int, int place, int row, int m, float v) { put(tile, place, row, m, v); });
            __syncwarp();
            if (s.lane == 0) barrier_arrive(&hand.empty);
        }
    }
}
// Floats of one buffer of sums: the warps', and a block's outputs where a cluster adds them up (all its warps share one set's k then).
template <int kRows, int kCount> constexpr int kSumsOf = (kWarps + 1) * kRows * kCount;

// One or two rows (w4_integer_kernel): products of whole numbers. An activation is fixed-point relative to the largest of its row and span, four signed 8-bit
// digits (30 bits and the sign), and each digit of each row is a column of m16n8k32: one row leaves seven of the eight columns of a product
// empty anyway. Codes are 8-bit operands after two masks and a shift for 8 of them, where 16-bit ones take nine instructions, and the
// instructions are what bounds this beside the memory. Sums of a span are exact in 32 bits:
//   sum (code - zero) X = sum code X - zero sum X,  |sum code X| <= 128 * 15 * 128,
// accumulated on 1.5 * 2^23's bits, so that the result is a float without a conversion. Scales of weights and activations are applied to
// that in fp32. An infinity or NaN makes its row's results NaN, and values below 2^-119 have no digits; a block that meets either in its
// outputs computes its part of the row again (plain_row).
constexpr int kDigits = 4, kIntegerRows = 2, kTopBit = 29, kLeast = -90;         // |X| < 2^(kTopBit + 1); least exponent of a span
constexpr uint32_t kIntegerBase = 0x4b400000u;                   // 12582912
// Whether an output tells that its row's activations have digits: it is finite and, unless it is 0, well above the least unit.
__device__ __forceinline__ bool has_digits(float v) { return v == 0.f || (fabsf(v) >= 7.8886090522101181e-31f && fabsf(v) <= 3.4028235e38f); }       // 2^-100

__device__ __forceinline__ void mma_integer(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// four values of a row from `at` on, zeros beyond k
__device__ __forceinline__ void load_four(const W4Params &p, int m, int at, float (&v)[4]) {
    const long long first = m * p.x_stride + at;
    const bool whole = p.vectors && at + 4 <= p.k;
    if (p.dtype == MSNH_B200_F32) {
        const float *x = static_cast<const float *>(p.x) + first;
        if (whole) {
            const float4 t = __ldg(reinterpret_cast<const float4 *>(x));
            v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = at + i < p.k ? x[i] : 0.f;
        }
    } else if (p.dtype == MSNH_B200_E4M3) {
        const uint8_t *x = static_cast<const uint8_t *>(p.x) + first;
        uint32_t raw = 0;
        if (whole) {
            raw = __ldg(reinterpret_cast<const uint32_t *>(x));
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) raw |= at + i < p.k ? static_cast<uint32_t>(x[i]) << (8 * i) : 0u;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __nv_fp8_e4m3 e;
            e.__x = static_cast<uint8_t>(raw >> (8 * i));
            v[i] = static_cast<float>(e);
        }
    } else {
        const uint16_t *x = static_cast<const uint16_t *>(p.x) + first;
        uint2 raw = make_uint2(0, 0);
        if (whole) {
            raw = __ldg(reinterpret_cast<const uint2 *>(x));
        } else {
            if (at < p.k) raw.x = x[0];
            if (at + 1 < p.k) raw.x |= static_cast<uint32_t>(x[1]) << 16;
            if (at + 2 < p.k) raw.y = x[2];
            if (at + 3 < p.k) raw.y |= static_cast<uint32_t>(x[3]) << 16;
        }
        if (p.dtype == MSNH_B200_F16) {
            __half2 h[2];
            memcpy(h, &raw, 8);
            const float2 a = __half22float2(h[0]), b = __half22float2(h[1]);
            v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
        } else {
            v[0] = __uint_as_float(raw.x << 16); v[1] = __uint_as_float(raw.x & 0xffff0000u);
            v[2] = __uint_as_float(raw.y << 16); v[3] = __uint_as_float(raw.y & 0xffff0000u);
        }
    }
}

// The digits of 128 values of a row, by a warp, a lane four of them. digits: [half unit][row][digit][4 x 16 bytes] in the order the lanes
// of the product read them; meta: [span][row][pair of digits] their sums and, twice, the activations' scale (16 bytes).
// `unit` counts from where the two begin, `at` is the first value's place in the row.
__device__ __forceinline__ void make_digits(const W4Params &p, int unit, int m, int at, int lane, uint8_t *digits, uint8_t *meta) {
    const int lanes = 32 / p.spans;
    float v[4];
    load_four(p, m, at + lane * 4, v);
    float top = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    bool finite = true;                                          // (a maximum drops NaN)
#pragma unroll
    for (int t = 0; t < 4; ++t) finite &= fabsf(v[t]) <= 3.4028235e38f;
    for (int o = 1; o < lanes; o *= 2) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
    const unsigned mask = lanes == 32 ? ~0u : (1u << lanes) - 1;
    finite = (__ballot_sync(~0u, finite) >> (lane / lanes * lanes) & mask) == mask;
    // (No unit is below 2^(kLeast - kTopBit), so that it and its products with scales are normal numbers. Values that are less than such a
    // unit become one of them: not 0, or nothing would show that they are there.)
    const int exponent = max(kLeast, static_cast<int>(__float_as_uint(top) >> 23) - 127);
    const float up = __uint_as_float(static_cast<uint32_t>(127 + kTopBit - exponent) << 23);
    const uint32_t unit_of = finite ? static_cast<uint32_t>(127 + exponent - kTopBit) << 23 : 0x7fffffffu;
    int x[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        x[t] = finite ? __float2int_rn(v[t] * up) : 0;
        if (exponent == kLeast && x[t] == 0 && v[t] != 0.f) x[t] = v[t] > 0.f ? 1 : -1;
    }
    const int in_half = lane * 4 % 64;
    uint8_t *const to = digits + (static_cast<size_t>(unit * 2 + lane / 16) * p.rows + m) * (kDigits * 64) + in_half % 32 / 8 * 16 + in_half / 32 * 8 + in_half % 8;
#pragma unroll
    for (int pair = 0; pair < kDigits / 2; ++pair) {
        int sums = 0;                                            // of two digits, 16 bits each: at most 128 * 128
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            uint32_t bytes = 0;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int digit = static_cast<int8_t>(x[t]);     // what is left is a multiple of 256 then
                bytes |= static_cast<uint32_t>(digit & 255) << (8 * t);
                x[t] = (x[t] - digit) >> 8;
                sums += digit << (16 * d);
            }
            *reinterpret_cast<uint32_t *>(to + (pair * 2 + d) * 64) = bytes;
        }
        for (int o = 1; o < lanes; o *= 2) sums += __shfl_xor_sync(~0u, sums, o);
        const int first = static_cast<int16_t>(sums);
        if (lane % lanes == 0)
            *reinterpret_cast<uint4 *>(meta + ((static_cast<size_t>(unit * p.spans + lane / lanes) * p.rows + m) * (kDigits / 2) + pair) * 16) =
                make_uint4(static_cast<uint32_t>(first), static_cast<uint32_t>((sums - first) >> 16), unit_of, unit_of);
    }
}

// Row m of the outputs of the block's tiles from the formula, value by value: for activations that have no digits. A warp an output; a lane
// eight values at a time, those of one word of the codes. Ten times as long as with digits (one such fp16 row times 8192 x 28672 346 us), for
// rows that no program lives on.
template <int kTiles> __device__ __noinline__ void plain_row(const W4Params &p, const Share<kTiles> &s, int m) {
    const int at = s.lane % 16, half = at / 8, quarter = at / 2 % 4, step = at % 2, in_unit = half * 64 + step * 32 + quarter * 8, record = p.wide ? 16 : 8;
    for (int i = s.from * kTileRows + s.warp; i < min(s.to * kTileRows, p.n); i += kWarps + kSummers) {
        const int row = i % kTileRows, pair = row % 8, high = row / 8;
        const uint8_t *tile = p.packed + static_cast<long long>(i / kTileRows) * p.units * p.unit_bytes;
        float sum = 0.f;
        for (int u = s.lane / 16; u < p.units; u += 2) {
            const uint8_t *unit = tile + u * p.unit_bytes, *span = unit + kCodeBytes + (in_unit / (kUnitK / p.spans) * 8 + pair) * record;
            const uint32_t word = *reinterpret_cast<const uint32_t *>(unit + half * 512 + (pair * 4 + quarter) * 16 + (2 * step + high) * 4);
            const float scale = p.wide ? reinterpret_cast<const float *>(span)[high] : __half2float(reinterpret_cast<const __half *>(span)[high]);
            const int zero = span[(p.wide ? 8 : 4) + high];
            float x[8];
            load_four(p, m, u * kUnitK + in_unit, *reinterpret_cast<float (*)[4]>(x));
            load_four(p, m, u * kUnitK + in_unit + 4, *reinterpret_cast<float (*)[4]>(x + 4));
#pragma unroll
            for (int v = 0; v < 8; ++v)
                if (u * kUnitK + in_unit + v < p.k) sum = fmaf(x[v], static_cast<float>(static_cast<int>(word >> (v % 4 * 8 + v / 4 * 4) & 15) - zero) * scale, sum);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
        if (s.lane == 0) store(p, m, i, sum);
    }
}

// All digits into the workspace, a warp 128 values of a row.
__global__ void w4_digits_kernel(const __grid_constant__ W4Params p) {
    pdl_enter();
    const int i = blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    if (i < p.units * p.rows) make_digits(p, i / p.rows, i % p.rows, i / p.rows * kUnitK, threadIdx.x % 32, p.digits_made, p.meta_made);
}

// Shared memory: sums, rings, digits, meta.
template <int kTiles, int kAhead>
__global__ void __launch_bounds__(kThreads, 1) w4_integer_kernel(const __grid_constant__ W4Params p) {
    constexpr int kRows = kTiles * kTileRows;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Handover hand;
    __shared__ int again[kIntegerRows];                          // rows that have no digits
    if (threadIdx.x == 0) {
        barrier_init(&hand.full, kWarps);
        barrier_init(&hand.empty, kSummers);
        again[0] = again[1] = 0;
    }
    auto cluster = cooperative_groups::this_cluster();
    const Share<kTiles> s(p, cluster.num_blocks(), cluster.block_rank());
    const uint32_t smem_at = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    if (!p.digits_made) pdl_enter();                             // (when the launch that makes them has begun, everything before it has ended)
    Units<kTiles, kAhead> units(p, s, smem_at + p.ring_at);
    const int lane = s.lane, half_digits = p.rows * kDigits * 64, span_meta = p.rows * kDigits * 8;
    if (p.digits_made) {
        const uint8_t *digits = p.digits_made + static_cast<size_t>(s.begin) * 2 * half_digits, *meta = p.meta_made + static_cast<size_t>(s.begin) * p.spans * span_meta;
        pdl_enter();
        for (int i = threadIdx.x * 16; i < s.block_units * 2 * half_digits; i += kThreads * 16) copy16(smem_at + p.x_at + i, digits + i);
        for (int i = threadIdx.x * 16; i < s.block_units * p.spans * span_meta; i += kThreads * 16) copy16(smem_at + p.meta_at + i, meta + i);
        copy_commit();
        copy_wait<0>();
    } else {
        for (int i = s.warp; i < s.block_units * p.rows; i += kWarps + kSummers)
            make_digits(p, i / p.rows, i % p.rows, (s.begin + i / p.rows) * kUnitK, lane, smem + p.x_at, smem + p.meta_at);
    }
    __syncthreads();
    // (columns beyond the rows' digits are the last one's again; their sums go nowhere)
    const uint32_t x_at = smem_at + p.x_at + 2 * (s.first - s.begin) * half_digits + min(lane / 4, p.rows * kDigits - 1) * 64 + lane % 4 * 16;
    const uint32_t meta_at = smem_at + p.meta_at + (s.first - s.begin) * p.spans * span_meta + min(lane % 4, p.rows * kDigits / 2 - 1) * 16;
    const int record = p.wide ? 16 : 8, span = 4 / p.spans;      // span: in steps of 32 values

    float acc[kTiles][4];
    const auto multiply = [&] {
        int part[kTiles][4];
#pragma unroll
        for (int r = 0; r < kTiles; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[r][i] = 0.f;
                part[r][i] = kIntegerBase;
            }
        uint32_t x_now = x_at, meta_now = meta_at;
#pragma unroll 1
        for (int u = 0; u < s.count; ++u) {
            units.wait();
            uint4 now[2][kTiles], x[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int r = 0; r < kTiles; ++r) now[half][r] = load_shared(units.slot + r * units.pitch + half * 512 + lane * 16);
                x[half] = load_shared(x_now);
                x_now += half_digits;
            }
#pragma unroll
            for (int step = 0; step < 4; ++step) {
                const int half = step / 2;
#pragma unroll
                for (int r = 0; r < kTiles; ++r) {
                    const uint32_t w0 = step % 2 ? now[half][r].z : now[half][r].x, w8 = step % 2 ? now[half][r].w : now[half][r].y;
                    const uint32_t a[4] = {w0 & 0x0f0f0f0fu, w8 & 0x0f0f0f0fu, w0 >> 4 & 0x0f0f0f0fu, w8 >> 4 & 0x0f0f0f0fu};
                    mma_integer(part[r], a, step % 2 ? x[half].z : x[half].x, step % 2 ? x[half].w : x[half].y);
                }
                if (step == 3 || (step == 1 && span <= 2) || span == 1) {
                    const uint4 meta = load_shared(meta_now);
                    const float unit_of = __uint_as_float(meta.z);
                    meta_now += span_meta;
#pragma unroll
                    for (int r = 0; r < kTiles; ++r) {
                        float2 scale;
                        uint32_t z0, z8;
                        take_record(units.slot + r * units.pitch + kCodeBytes + (step / span * 8 + lane / 4) * record, p.wide, scale, z0, z8);
                        const float factor[2] = {scale.x * unit_of, scale.y * unit_of};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int sum = part[r][i] - static_cast<int>(i < 2 ? z0 : z8) * static_cast<int>(i % 2 ? meta.y : meta.x);
                            acc[r][i] = fmaf(factor[i / 2], __int_as_float(sum) - 12582912.f, acc[r][i]);
                            part[r][i] = kIntegerBase;
                        }
                    }
                }
            }
            units.next();
        }
    };
    // lanes 4 i and 4 i + 2 have digits 0 and 1 of the two rows, their neighbours 2 and 3
    const auto leave = [&](float *to) {
#pragma unroll
        for (int r = 0; r < kTiles; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float v = fmaf(acc[r][2 * i + 1], 256.f, acc[r][2 * i]);
                v = fmaf(__shfl_down_sync(~0u, v, 1), 65536.f, v);
                if (lane % 2 == 0) to[lane % 4 / 2 * kRows + r * kTileRows + lane / 4 + i * 8] = v;
            }
    };
    turns<kTiles, kIntegerRows>(p, s, cluster, reinterpret_cast<float *>(smem), hand, multiply, leave, [&](int m, float v) { if (!has_digits(v)) again[m] = 1; });
    copy_wait<0>();
    __syncthreads();
#pragma unroll 1
    for (int m = 0; m < p.rows; ++m)
        if (again[m]) plain_row<kTiles>(p, s, m);
}

// The activations at place i of the 16-bit operands, [step of 32 values][row][4 x 16 bytes], from unit `begin` on.
template <typename X> __device__ __forceinline__ void load_raw(const W4Params &p, int begin, int i, Raw<X> &raw) {
    const int m = i / 4 % p.rows, at = (begin * 4 + i / 4 / p.rows) * 32 + i % 4 * 8;
    const X *row = static_cast<const X *>(p.x) + m * p.x_stride + at;
    if (p.vectors && at + 8 <= p.k) raw.load(row);
    else raw.load(row, p.k - at);
}

// All of them into the workspace, [part] first.
template <typename X> __global__ void w4_operands_kernel(const __grid_constant__ W4Params p) {
    pdl_enter();
    const int i = blockIdx.x * blockDim.x + threadIdx.x, all = p.units * p.rows * 16;
    if (i >= all) return;
    Raw<X> raw;
    load_raw<X>(p, 0, i, raw);
    uint32_t b[Operand<X>::kParts][4];
    raw.operands(b);
#pragma unroll
    for (int part = 0; part < Operand<X>::kParts; ++part)
        reinterpret_cast<uint4 *>(p.digits_made)[static_cast<size_t>(part) * all + i] = make_uint4(b[part][0], b[part][1], b[part][2], b[part][3]);
}

// More rows: rows of the weights are the 16 rows of m16n8k16, activations its columns. Operands of the codes less zero point are made in
// registers (exact); a span's products are summed on the tensor cores and its scale is applied to that sum in fp32.
// The activations, as operands in the order the lanes read them, are made by a launch before this one, or by every block where there are
// few. kStaged: they are in shared memory; otherwise they are read from the workspace (the caches) for every tile.
template <typename X, int kColumns, int kTiles, int kAhead, bool kStaged>
__global__ void __launch_bounds__(kThreads, 1) w4_linear_kernel(const __grid_constant__ W4Params p) {
    using H = typename Operand<X>::Type;
    constexpr int kParts = Operand<X>::kParts, kRows = kTiles * kTileRows;
    extern __shared__ __align__(16) uint8_t smem[];              // sums, rings, activations [part][step of 32 values][row][4 x 16 bytes]
    __shared__ Handover hand;
    if (threadIdx.x == 0) {
        barrier_init(&hand.full, kWarps);
        barrier_init(&hand.empty, kSummers);
    }
    auto cluster = cooperative_groups::this_cluster();
    const Share<kTiles> s(p, cluster.num_blocks(), cluster.block_rank());
    const uint32_t smem_at = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    if (!p.digits_made) pdl_enter();                             // (when the launch that makes them has begun, everything before it has ended)
    Units<kTiles, kAhead> units(p, s, smem_at + p.ring_at);
    const int lane = s.lane, part_pitch = 4 * s.block_units * p.rows * 64;
    if (kStaged) {
        if (p.digits_made) {
            pdl_enter();
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                const uint8_t *from = p.digits_made + (static_cast<size_t>(part) * p.units + s.begin) * p.rows * 256;
                for (int i = threadIdx.x * 16; i < part_pitch; i += kThreads * 16) copy16(smem_at + p.x_at + part * part_pitch + i, from + i);
            }
            copy_commit();
            copy_wait<0>();
        } else {
            // (four places of a thread at a time, so that their reads are under way together)
            constexpr int kBatch = 4;
            for (int base = threadIdx.x; base < part_pitch / 16; base += kBatch * kThreads) {
                Raw<X> raw[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; ++j)
                    if (base + j * kThreads < part_pitch / 16) load_raw<X>(p, s.begin, base + j * kThreads, raw[j]);
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int i = base + j * kThreads;
                    if (i >= part_pitch / 16) break;
                    uint32_t b[kParts][4];
                    raw[j].operands(b);
#pragma unroll
                    for (int part = 0; part < kParts; ++part)
                        *reinterpret_cast<uint4 *>(smem + p.x_at + part * part_pitch + i * 16) = make_uint4(b[part][0], b[part][1], b[part][2], b[part][3]);
                }
            }
        }
    } else {
        pdl_enter();
    }
    __syncthreads();
    // (a column beyond the rows is the last row again; its sums are not stored)
    const int record = p.wide ? 16 : 8, span = 4 / p.spans;      // span: in steps of 32 values
    const uint32_t staged_at = smem_at + p.x_at + (4 * (s.first - s.begin) * p.rows * 4 + lane % 4) * 16;
    float acc[kTiles][kColumns][4];
    const auto multiply = [&] {
        float part[kTiles][kColumns][4] = {};
#pragma unroll
        for (int r = 0; r < kTiles; ++r)
#pragma unroll
            for (int c = 0; c < kColumns; ++c) acc[r][c][0] = acc[r][c][1] = acc[r][c][2] = acc[r][c][3] = 0.f;
        uint32_t x_now = staged_at;
        int step_now = s.first * 4;
        float2 scale[kTiles];
        Zero<H> zero[kTiles][2];
#pragma unroll 1
        for (int u = 0; u < s.count; ++u) {
            units.wait();
#pragma unroll
            for (int step = 0; step < 4; ++step) {
                uint32_t a[kTiles][2][4];
#pragma unroll
                for (int r = 0; r < kTiles; ++r) {
                    const uint32_t at = units.slot + r * units.pitch;
                    if (step == 0 || (step == 2 && span <= 2) || span == 1) {
                        uint32_t z0, z8;
                        take_record(at + kCodeBytes + (step / span * 8 + lane / 4) * record, p.wide, scale[r], z0, z8);
                        zero[r][0].set(z0);
                        zero[r][1].set(z8);
                    }
                    uint2 now;
                    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(now.x), "=r"(now.y) : "r"(at + step / 2 * 512 + lane * 16 + step % 2 * 8) : "memory");
                    uint32_t low[4], high[4];
                    zero[r][0].operand(now.x, p.exponents, low);
                    zero[r][1].operand(now.y, p.exponents, high);
#pragma unroll
                    for (int i = 0; i < 2; ++i) { a[r][i][0] = low[2 * i]; a[r][i][1] = high[2 * i]; a[r][i][2] = low[2 * i + 1]; a[r][i][3] = high[2 * i + 1]; }
                }
#pragma unroll
                for (int c = 0; c < kColumns; ++c) {
                    const int m = min(c * 8 + lane / 4, p.rows - 1);
                    uint32_t b[kParts][4];
                    if (kStaged) {
#pragma unroll
                        for (int i = 0; i < kParts; ++i) {
                            const uint4 v = load_shared(x_now + m * 64 + i * part_pitch);
                            memcpy(b[i], &v, 16);
                        }
                    } else {
                        const uint4 *from = reinterpret_cast<const uint4 *>(p.digits_made) + (static_cast<size_t>(step_now) * p.rows + m) * 4 + lane % 4;
#pragma unroll
                        for (int i = 0; i < kParts; ++i) {
                            const uint4 v = __ldg(from + static_cast<size_t>(i) * p.units * p.rows * 16);
                            memcpy(b[i], &v, 16);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kParts; ++i)
#pragma unroll
                        for (int r = 0; r < kTiles; ++r) {
                            mma<H>(part[r][c], a[r][0], b[i][0], b[i][1]);
                            mma<H>(part[r][c], a[r][1], b[i][2], b[i][3]);
                        }
                }
                x_now += p.rows * 64;
                ++step_now;
                if (step == 3 || (step == 1 && span <= 2) || span == 1)
#pragma unroll
                    for (int r = 0; r < kTiles; ++r)
#pragma unroll
                        for (int c = 0; c < kColumns; ++c)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                acc[r][c][i] = fmaf(i < 2 ? scale[r].x : scale[r].y, part[r][c][i], acc[r][c][i]);
                                part[r][c][i] = 0.f;
                            }
            }
            units.next();
        }
    };
    const auto leave = [&](float *to) {
#pragma unroll
        for (int r = 0; r < kTiles; ++r)
#pragma unroll
            for (int c = 0; c < kColumns; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) to[(c * 8 + lane % 4 * 2 + i % 2) * kRows + r * kTileRows + lane / 4 + i / 2 * 8] = acc[r][c][i] * Zero<H>::kUnit;
    };
    turns<kTiles, kColumns * 8>(p, s, cluster, reinterpret_cast<float *>(smem), hand, multiply, leave, [](int, float) {});
    copy_wait<0>();
}

// Still more rows, whose activations no block has room for and every tile would read again from the caches: a warp has a tile to itself, and
// the block's warps go through k together, each unit's activations copied once for all of them, a ring ahead like the weights. Where that
// leaves SMs without a block, the blocks of a cluster share k.
// 64 fp16 rows times 8192 x 8192 take 43.5 us (197 TFLOP/s) where reading them from the caches for every tile took 100; times 4096 x 4096
// 25.6 (40 before). Of the 2.2 us of a unit the products are 1.1 and the reads of the activations' operands from shared memory another 1.1:
// tcgen05 would need the weights as operands in shared memory, scaled before they are summed or unloaded for every group.
template <typename X, int kColumns, int kAhead>
__global__ void __launch_bounds__(kWarps * 32, 1) w4_rows_kernel(const __grid_constant__ W4Params p) {
    using H = typename Operand<X>::Type;
    constexpr int kParts = Operand<X>::kParts, kCount = kColumns * 8, kThreads = kWarps * 32;
    extern __shared__ __align__(16) uint8_t smem[];              // the weights' rings, the activations' [stage][part][step of 32 values][row][4 x 16 bytes]
    auto cluster = cooperative_groups::this_cluster();
    const Share<1> s(p, cluster.num_blocks(), cluster.block_rank());
    const uint32_t smem_at = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    Units<1, kAhead> units(p, s, smem_at + p.ring_at);
    const int lane = s.lane, part_bytes = p.rows * 256, stage_bytes = kParts * part_bytes;
    const int all = (s.to - s.from + s.turn - 1) / s.turn * s.block_units;      // units of all turns
    int issued = 0, next = 0, fill = 0, stage = 0;
    const auto copy_x = [&] {
        if (issued < all) {
#pragma unroll
            for (int part = 0; part < kParts; ++part) {
                const uint8_t *from = p.digits_made + (static_cast<size_t>(part) * p.units + s.begin + next) * part_bytes;
                const uint32_t to = smem_at + p.x_at + fill * stage_bytes + part * part_bytes;
                for (int i = threadIdx.x * 16; i < part_bytes; i += kThreads * 16) copy16(to + i, from + i);
            }
        }
        ++issued;
        next = next + 1 == s.block_units ? 0 : next + 1;
        fill = fill == kAhead - 1 ? 0 : fill + 1;
    };
    pdl_enter();
#pragma unroll 1
    for (int i = 0; i < kAhead - 1; ++i) copy_x();
    copy_commit();
    copy_wait<0>();                                              // (from here on a group a unit)
    const int record = p.wide ? 16 : 8, span = 4 / p.spans;      // span: in steps of 32 values
    float acc[kColumns][4];
    for (int tile = s.mine, first = s.from; first < s.to; first += s.turn, tile += s.turn) {
        float part[kColumns][4] = {};
        float2 scale;
        Zero<H> zero[2];
#pragma unroll
        for (int c = 0; c < kColumns; ++c) acc[c][0] = acc[c][1] = acc[c][2] = acc[c][3] = 0.f;
#pragma unroll 1
        for (int u = 0; u < s.block_units; ++u) {
            copy_wait<kAhead - 2>();
            __syncthreads();                                     // (everybody's copies; the stage that is filled next has been read)
            copy_x();
            units.copy();
            if (tile < s.to) {
                uint32_t x_now = smem_at + p.x_at + stage * stage_bytes + lane % 4 * 16;
#pragma unroll
                for (int step = 0; step < 4; ++step) {
                    if (step == 0 || (step == 2 && span <= 2) || span == 1) {
                        uint32_t z0, z8;
                        take_record(units.slot + kCodeBytes + (step / span * 8 + lane / 4) * record, p.wide, scale, z0, z8);
                        zero[0].set(z0);
                        zero[1].set(z8);
                    }
                    uint2 now;
                    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(now.x), "=r"(now.y) : "r"(units.slot + step / 2 * 512 + lane * 16 + step % 2 * 8) : "memory");
                    uint32_t low[4], high[4], a[2][4];
                    zero[0].operand(now.x, p.exponents, low);
                    zero[1].operand(now.y, p.exponents, high);
#pragma unroll
                    for (int i = 0; i < 2; ++i) { a[i][0] = low[2 * i]; a[i][1] = high[2 * i]; a[i][2] = low[2 * i + 1]; a[i][3] = high[2 * i + 1]; }
#pragma unroll
                    for (int c = 0; c < kColumns; ++c) {
                        const int m = min(c * 8 + lane / 4, p.rows - 1);        // (a column beyond the rows is the last row again)
#pragma unroll
                        for (int i = 0; i < kParts; ++i) {
                            const uint4 b = load_shared(x_now + m * 64 + i * part_bytes);
                            mma<H>(part[c], a[0], b.x, b.y);
                            mma<H>(part[c], a[1], b.z, b.w);
                        }
                    }
                    x_now += p.rows * 64;
                    if (step == 3 || (step == 1 && span <= 2) || span == 1)
#pragma unroll
                        for (int c = 0; c < kColumns; ++c)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                acc[c][i] = fmaf(i < 2 ? scale.x : scale.y, part[c][i], acc[c][i]);
                                part[c][i] = 0.f;
                            }
                }
            }
            units.next();
            stage = stage == kAhead - 1 ? 0 : stage + 1;
        }
        if (s.ranks == 1 && tile < s.to)
#pragma unroll
            for (int c = 0; c < kColumns; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int m = c * 8 + lane % 4 * 2 + i % 2, row = tile * kTileRows + lane / 4 + i / 2 * 8;
                    if (m < p.rows && row < p.n) store(p, m, row, acc[c][i] * Zero<H>::kUnit);
                }
    }
    copy_wait<0>();
    if (s.ranks == 1) return;
    // (one turn then: the sums take the rings' place, [warp][column][row])
    __syncthreads();
    float *const sums = reinterpret_cast<float *>(smem);
#pragma unroll
    for (int c = 0; c < kColumns; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[(s.warp * kCount + c * 8 + lane % 4 * 2 + i % 2) * kTileRows + lane / 4 + i / 2 * 8] = acc[c][i] * Zero<H>::kUnit;
    cluster.sync();
    for (int o = s.rank * kThreads + threadIdx.x; o < kWarps * p.rows * (kTileRows / 4); o += s.ranks * kThreads) {
        const int set = o / (p.rows * (kTileRows / 4)), m = o / (kTileRows / 4) % p.rows, quarter = o % (kTileRows / 4);
        if (s.from + set >= s.to) continue;
        float4 v[kMostRanks];                                    // (all reads are under way before the first is added)
#pragma unroll
        for (int q = 0; q < kMostRanks; ++q)
            if (q < s.ranks) v[q] = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(&sums[(set * kCount + m) * kTileRows + quarter * 4], q));
#pragma unroll
        for (int q = 1; q < kMostRanks; ++q)
            if (q < s.ranks) { v[0].x += v[q].x; v[0].y += v[q].y; v[0].z += v[q].z; v[0].w += v[q].w; }
        const int row = (s.from + set) * kTileRows + quarter * 4;
        if (row < p.n) store(p, m, row, v[0].x);
        if (row + 1 < p.n) store(p, m, row + 1, v[0].y);
        if (row + 2 < p.n) store(p, m, row + 2, v[0].z);
        if (row + 3 < p.n) store(p, m, row + 3, v[0].w);
    }
    cluster.sync();                                              // (no block ends while another reads its sums)
}

constexpr size_t kSmemMost = 224 * 1024;                         // of shared memory for a block

template <typename Kernel>
cudaError_t launch(const MsnhB200Ctx *ctx, Kernel kernel, std::atomic<uint64_t> &done, const W4Params &p, int blocks, int ranks, int threads, size_t smem, bool dependent, void *stream) {
    // the attribute is a kernel's and a device's: set by the first call there
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (!(done.load(std::memory_order_acquire) & bit)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMost));
        if (e != cudaSuccess) return e;
        done.fetch_or(bit, std::memory_order_release);
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks * ranks);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = dependent ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, p);
}

// Clusters of `ranks` blocks, a block an SM, that the device holds at the same time: fewer than SMs / ranks, since a cluster lies in one
// part of the device (74, 33 and 15 of 2, 4 and 8 blocks; one cluster more runs after all the others). Asked for once.
int clusters_at_once(const MsnhB200Ctx *ctx, int ranks) {
    static std::atomic<int> known[64][4];
    if (ranks == 1) return ctx->sm_count;
    std::atomic<int> &place = known[ctx->device & 63][ranks == 2 ? 1 : ranks == 4 ? 2 : 3];
    int n = place.load(std::memory_order_relaxed);
    if (n) return n;
    const auto kernel = w4_linear_kernel<__half, 1, 1, 5, true>;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(ranks);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kSmemMost;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMost)) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &config) != cudaSuccess || n < 1) {
        cudaGetLastError();                                      // (a cluster less than would fit costs time only)
        n = std::max(1, ctx->sm_count / ranks * 3 / 4);
    }
    place.store(n, std::memory_order_relaxed);
    return n;
}

// How many warps of a block share a tile's k, `tiles` at a time: what takes the fewest units one after the other in the busiest warp (turns x
// units of each), the more the better at the same count; and the turns of that block.
struct Split { int warps, turns; };
Split split_of(const MsnhB200Ctx *ctx, const W4Params &p, int tiles) {
    const auto up = [](int a, int b) { return (a + b - 1) / b; };
    const auto turns = [&](int split) {
        const int per_turn = kWarps / split * tiles;
        return up(up(p.tiles, std::min(up(p.tiles, per_turn), ctx->sm_count)), per_turn);
    };
    const auto cost = [&](int split) { return static_cast<long long>(turns(split)) * up(p.units, split); };
    int best = 1;
    for (int split = 2; split <= kWarps && split <= p.units; split *= 2)
        if (cost(split) <= cost(best)) best = split;
    return {best, turns(best)};
}

// How a launch is cut up: warps as above. Where that leaves SMs without a block, a cluster shares it further, down to two units
// of k a warp; and where that is what makes room for the activations (x_bytes: of those of some units). (A cluster has room for the outputs of one
// set of warps.) Returns whether there is room.
template <typename Bytes>
bool share_out(const MsnhB200Ctx *ctx, W4Params &p, int tiles, Bytes x_bytes, int &ranks, int &blocks) {
    const auto up = [](int a, int b) { return (a + b - 1) / b; };
    p.split = split_of(ctx, p, tiles).warps;
    const int turns = up(p.tiles, kWarps / p.split * tiles);
    const auto units = [&] { return std::min(p.units, p.split * up(p.units, p.split * ranks)); };
    ranks = 1;
    while (p.split == kWarps && ranks < kMostRanks && turns <= clusters_at_once(ctx, ranks * 2) && p.split * ranks * 4 <= p.units) ranks *= 2;
    const int wanted = ranks;
    while (p.split == kWarps && ranks < kMostRanks && p.x_at + x_bytes(units()) > kSmemMost && p.split * ranks * 2 <= p.units) ranks *= 2;
    const bool room = p.x_at + x_bytes(units()) <= kSmemMost;
    if (!room) ranks = wanted;
    p.share = up(p.units, p.split * ranks);
    p.block_units = units();
    blocks = std::min(turns, clusters_at_once(ctx, ranks));
    return room;
}

// Digits are made by every block for itself, or, where that is over kOwnDigits turns of its warps (1 us each), by a launch before it: one and
// two rows times 8192 x 28672 28.2 and 29.1 us, by every block 31.3 and 37.0; times 2048 x 40000, which is below, 14.8 and 19.3 against 16.0
// and 19.1 apart.
constexpr int kOwnDigits = 2;
size_t digit_bytes(int rows, int units) { return static_cast<size_t>(units) * 2 * rows * kDigits * 64; }
size_t meta_bytes(int rows, int units, int spans) { return static_cast<size_t>(units) * spans * rows * kDigits * 8; }
bool digits_apart(int rows, int units) { return rows <= kIntegerRows && rows * units > kOwnDigits * (kWarps + kSummers); }
// 16-bit operands are made by every block where they are at most kOwnOperands bytes, which find room beside the sums and rings of every
// kernel (86 KB at least); a launch before it makes more than that, and blocks without room for them read them from the workspace. (Seven
// rows times 4096 x 4096 and 5120 x 13824: 8.8 and 17.6 us by every block, 10.6 and 19.7 apart.)
constexpr size_t kOwnOperands = 80 * 1024;
size_t operand_bytes(int rows, int dtype, int units) { return static_cast<size_t>(dtype == MSNH_B200_F32 ? 3 : 1) * units * rows * 256; }
bool operands_apart(int rows, int dtype, int units) { return operand_bytes(rows, dtype, units) > kOwnOperands; }

template <int kTiles, int kAhead>
bool launch_integer(const MsnhB200Ctx *ctx, W4Params p, void *stream, cudaError_t &e) {
    p.ring_at = kSumsOf<kTiles * kTileRows, kIntegerRows> * 4;
    p.x_at = p.ring_at + kWarps * kAhead * kTiles * static_cast<int>(p.unit_bytes);
    const auto bytes = [&](int units) { return digit_bytes(p.rows, units) + meta_bytes(p.rows, units, p.spans); };
    int ranks, blocks;
    if (!share_out(ctx, p, kTiles, bytes, ranks, blocks)) return false;
    p.meta_at = p.x_at + static_cast<int>(digit_bytes(p.rows, p.block_units));
    if (p.digits_made) {
        p.meta_made = p.digits_made + digit_bytes(p.rows, p.units);
        e = launch_token_kernel(w4_digits_kernel, dim3((p.units * p.rows + 3) / 4), 128, 0, stream, ctx->pdl, p);
        if (e != cudaSuccess) return true;
    }
    static std::atomic<uint64_t> done{0};
    e = launch(ctx, w4_integer_kernel<kTiles, kAhead>, done, p, blocks, ranks, kThreads, p.x_at + bytes(p.block_units), ctx->pdl, stream);
    return true;
}

template <typename X, int kColumns, int kTiles, int kAhead>
cudaError_t launch(const MsnhB200Ctx *ctx, W4Params p, void *stream) {
    p.ring_at = kSumsOf<kTiles * kTileRows, kColumns * 8> * 4;
    p.x_at = p.ring_at + kWarps * kAhead * kTiles * static_cast<int>(p.unit_bytes);
    p.exponents = Zero<typename Operand<X>::Type>::kExponents;
    const auto bytes = [&](int units) { return static_cast<size_t>(Operand<X>::kParts) * 4 * units * p.rows * 64; };
    int ranks, blocks;
    const bool staged = share_out(ctx, p, kTiles, bytes, ranks, blocks);
    if (!operands_apart(p.rows, p.dtype, p.units)) p.digits_made = nullptr;
    if (!staged && !p.digits_made) return cudaErrorInvalidConfiguration;         // (there is nothing to read them from)
    if (p.digits_made) {
        const cudaError_t e = launch_token_kernel(w4_operands_kernel<X>, dim3((p.units * p.rows * 16 + 127) / 128), 128, 0, stream, ctx->pdl, p);
        if (e != cudaSuccess) return e;
    }
    static std::atomic<uint64_t> done[2];
    return staged ? launch(ctx, w4_linear_kernel<X, kColumns, kTiles, kAhead, true>, done[0], p, blocks, ranks, kThreads, p.x_at + bytes(p.block_units), ctx->pdl, stream)
                  : launch(ctx, w4_linear_kernel<X, kColumns, kTiles, kAhead, false>, done[1], p, blocks, ranks, kThreads, p.x_at, ctx->pdl, stream);
}

template <typename X, int kColumns, int kAhead>
cudaError_t launch_rows(const MsnhB200Ctx *ctx, W4Params p, void *stream) {
    const int turns = (p.tiles + kWarps - 1) / kWarps;
    int ranks = 1;
    while (ranks < kMostRanks && turns <= clusters_at_once(ctx, ranks * 2) && ranks * 2 <= p.units) ranks *= 2;
    p.split = 1;
    p.share = (p.units + ranks - 1) / ranks;
    p.block_units = p.share;
    p.ring_at = 0;
    p.x_at = kWarps * kAhead * static_cast<int>(p.unit_bytes);
    p.exponents = Zero<typename Operand<X>::Type>::kExponents;
    const cudaError_t e = launch_token_kernel(w4_operands_kernel<X>, dim3((p.units * p.rows * 16 + 127) / 128), 128, 0, stream, ctx->pdl, p);
    if (e != cudaSuccess) return e;
    const size_t rings = p.x_at + static_cast<size_t>(kAhead) * Operand<X>::kParts * p.rows * 256, sums = static_cast<size_t>(kWarps) * kTileRows * kColumns * 8 * 4;
    static std::atomic<uint64_t> done{0};
    return launch(ctx, w4_rows_kernel<X, kColumns, kAhead>, done, p, std::min(turns, clusters_at_once(ctx, ranks)), ranks, kWarps * 32, std::max(rings, ranks > 1 ? sums : 0), ctx->pdl, stream);
}

// Whole numbers for one and two rows of many tiles, two tiles at a time, where their longer preparation is worth it: for 16- and 8-bit
// activations one row from 4 tiles an SM and k of 2048 on, two rows from 5 and 4096, and from 4 where a block is through in one turn with
// them and not without; for fp32 ones, which are three operands otherwise, from 4 tiles on whatever k. us in whole numbers / with 16-bit
// operands (8-bit and bf16 activations as fp16 within 3 %):
//                    1 row fp16     fp32           2 rows fp16    fp32
//     512 x 12288    4.7 / 4.9      4.7 / 5.6      5.3 / 5.8      5.2 / 6.5       (one turn against two)
//     512 x 40000    9.5 / 8.9      9.5 / 9.9      12.8 / 11.2    12.7 / 12.3     (three against five)
//     768 x 16000    5.6 / 4.9                     6.1 / 5.2                      (one of either)
//     1024 x 9600    6.5 / 5.6      6.4 / 6.5      7.8 / 6.2      7.8 / 7.0
//     1024 x 40000   11.6 / 12.0    11.6 / 14.1    14.5 / 14.3    14.6 / 16.0
//     2048 x 9600    7.5 / 7.8      7.5 / 9.2      10.0 / 7.9     9.9 / 9.3
//     2048 x 20000   10.2 / 12.1    10.2 / 14.0    13.3 / 12.2    13.3 / 14.3
//     2048 x 40000   14.8 / 19.8    14.8 / 22.7    19.3 / 20.1    19.2 / 23.0
//     4096 x 9600    11.3 / 10.7    11.3 / 14.0    11.9 / 10.8    11.9 / 14.5
//     4096 x 12288   11.6 / 12.1    11.7 / 15.9    12.3 / 12.2    12.2 / 16.4
//     4096 x 20000   14.5 / 15.9    14.5 / 21.5    15.7 / 16.0    15.7 / 21.9
//     8192 x 28672   28.1 / 34.1    28.2 / 49.8    28.9 / 34.4    29.0 / 53.8
// (times 4096 x 4096 one fp16 row took 7.5 in whole numbers, 6.2 with operands.)
// Nine to sixteen rows keep their activations in shared memory where tiles are few, so that all warps of a block can share k (nine fp16 rows
// times 4096 x 4096 10.1 us against 14.1; sixteen times 4096 x 12288 and 8192 x 28672 29.8 and 105 us against 22.7 and 68).
template <typename X>
cudaError_t launch(const MsnhB200Ctx *ctx, const W4Params &p, void *stream) {
    if (p.rows <= kIntegerRows && p.tiles >= 4 * ctx->sm_count &&
        (std::is_same<X, float>::value || (p.tiles >= (3 + p.rows) * ctx->sm_count && p.units >= 16 * p.rows) ||
         (split_of(ctx, p, 2).turns == 1 && split_of(ctx, p, 1).turns > 1))) {
        cudaError_t e = cudaSuccess;
        W4Params digits = p;
        if (!digits_apart(p.rows, p.units)) digits.digits_made = nullptr;
        if (launch_integer<2, 3>(ctx, digits, stream, e)) return e;
    }
    if (p.rows <= 8) return launch<X, 1, 1, 5>(ctx, p, stream);
    if (p.rows <= 16) return p.tiles >= 4 * ctx->sm_count ? launch_rows<X, 2, 4>(ctx, p, stream) : launch<X, 2, 1, 4>(ctx, p, stream);
    if (p.rows <= 32) return launch_rows<X, 4, 4>(ctx, p, stream);
    if (p.rows <= 48) return launch_rows<X, 6, 3>(ctx, p, stream);
    return launch_rows<X, 8, 3>(ctx, p, stream);
}

size_t workspace_of(const W4Layout &l, const MsnhB200W4Linear &a) {
    if (a.rows < 1) return 0;
    const size_t digits = digits_apart(a.rows, l.units) ? digit_bytes(a.rows, l.units) + meta_bytes(a.rows, l.units, l.spans) : 0;
    return std::max(digits, a.rows > 8 || operands_apart(a.rows, a.dtype, l.units) ? operand_bytes(a.rows, a.dtype, l.units) : 0);
}

constexpr int kMostOutputs = 1 << 30, kMostValues = 1 << 27;
int check_weights(MsnhB200Ctx *ctx, const MsnhB200W4 *w, const char *what) {
    if (w->n < 1 || w->k < 1) return fail(ctx, MSNH_B200_ERR_ARG, "%s: %d x %d weights", what, w->n, w->k);
    // (64 rows times 16 pieces of k / 128 units are counted in 32 bits)
    if (w->n > kMostOutputs || w->k > kMostValues) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: %d x %d weights (at most 2^30 x 2^27 are taken)", what, w->n, w->k);
    if (w->group < 32 || w->group % 32) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: groups of %d values (a multiple of 32 is wanted)", what, w->group);
    if (!is_float_type(w->scale_dtype)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "%s: scales of type %d", what, w->scale_dtype);
    return MSNH_B200_OK;
}

template <typename S, typename Out>
cudaError_t launch_pack_records(const W4Layout &l, const void *scales, const uint8_t *zeros, uint8_t *packed, void *stream) {
    const long long count = static_cast<long long>(l.tiles) * l.units * l.spans * 8;
    const unsigned grid = static_cast<unsigned>(std::min<long long>((count + 255) / 256, 148 * 16));
    return launch_token_kernel(w4_pack_records_kernel<S, Out>, dim3(grid), 256, 0, stream, false, static_cast<const S *>(scales), zeros, l.n, l.k, l.units,
                               l.spans, l.group, l.groups, l.unit_bytes, count, packed);
}

}  // namespace
}  // namespace msnh

using namespace msnh;

extern "C" {

int msnh_b200_w4_pack_bytes(MsnhB200Ctx *ctx, const MsnhB200W4 *w, size_t *bytes) try {
    if (!ctx || !w || !bytes) return MSNH_B200_ERR_ARG;
    if (const int rc = check_weights(ctx, w, "w4_pack_bytes")) return rc;
    *bytes = W4Layout(*w).bytes;
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_w4_pack(MsnhB200Ctx *ctx, const MsnhB200W4 *w, const uint8_t *codes, int64_t codes_stride, const void *scales, const uint8_t *zeros,
                      void *packed, void *stream) try {
    if (!ctx || !w) return MSNH_B200_ERR_ARG;
    if (const int rc = check_weights(ctx, w, "w4_pack")) return rc;
    if (!codes || !scales || !packed) return fail(ctx, MSNH_B200_ERR_ARG, "w4_pack: null codes, scales or packed");
    if ((w->has_zeros != 0) != (zeros != nullptr)) return fail(ctx, MSNH_B200_ERR_ARG, "w4_pack: has_zeros says whether there are zeros");
    if (!aligned16(packed)) return fail(ctx, MSNH_B200_ERR_ARG, "w4_pack: packed is not 16-byte aligned");
    if (codes_stride < 0) return fail(ctx, MSNH_B200_ERR_ARG, "w4_pack: codes_stride is negative");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    const W4Layout l(*w);
    uint8_t *out = static_cast<uint8_t *>(packed);
    const long long words = static_cast<long long>(l.tiles) * l.units * (kCodeBytes / 4);
    const unsigned grid = static_cast<unsigned>(std::min<long long>((words + 255) / 256, 148 * 32));
    CUDA_TRY(ctx, launch_token_kernel(w4_pack_codes_kernel, dim3(grid), 256, 0, stream, false, codes, codes_stride, l.n, l.k, l.units, l.unit_bytes, words, out));
    CUDA_TRY(ctx, w->scale_dtype == MSNH_B200_F16  ? (launch_pack_records<__half, __half>(l, scales, zeros, out, stream))
                : w->scale_dtype == MSNH_B200_BF16 ? (launch_pack_records<__nv_bfloat16, float>(l, scales, zeros, out, stream))
                                                   : (launch_pack_records<float, float>(l, scales, zeros, out, stream)));
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_w4_linear_workspace(MsnhB200Ctx *ctx, const MsnhB200W4 *w, const MsnhB200W4Linear *a, size_t *bytes) try {
    if (!ctx || !w || !a || !bytes) return MSNH_B200_ERR_ARG;
    if (const int rc = check_weights(ctx, w, "w4_linear_workspace")) return rc;
    *bytes = workspace_of(W4Layout(*w), *a);
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

int msnh_b200_w4_linear(MsnhB200Ctx *ctx, const MsnhB200W4 *w, const MsnhB200W4Linear *a, void *stream) try {
    if (!ctx || !w || !a) return MSNH_B200_ERR_ARG;
    if (const int rc = check_weights(ctx, w, "w4_linear")) return rc;
    if (a->rows < 0 || a->rows > MSNH_B200_W4_MAX_ROWS) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "w4_linear: %d rows (at most %d)", a->rows, MSNH_B200_W4_MAX_ROWS);
    if (!is_float_type(a->dtype) && a->dtype != MSNH_B200_E4M3) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "w4_linear: x of type %d", a->dtype);
    if (!is_float_type(a->out_dtype)) return fail(ctx, MSNH_B200_ERR_UNSUPPORTED, "w4_linear: y of type %d", a->out_dtype);
    if (a->rows == 0) return MSNH_B200_OK;
    if (!a->x || !a->y || !w->packed) return fail(ctx, MSNH_B200_ERR_ARG, "w4_linear: null x, y or weights");
    if (!aligned16(w->packed)) return fail(ctx, MSNH_B200_ERR_ARG, "w4_linear: the packed weights are not 16-byte aligned");
    if (a->x_stride < 0 || a->y_stride < (a->rows > 1 ? w->n : 0)) return fail(ctx, MSNH_B200_ERR_ARG, "w4_linear: rows overlap");
    DeviceScope scope(ctx->device);
    CUDA_TRY(ctx, scope.status);
    const W4Layout l(*w);
    const size_t wanted = workspace_of(l, *a);
    if (wanted && (!a->workspace || a->workspace_bytes < wanted || !aligned16(a->workspace)))
        return fail(ctx, MSNH_B200_ERR_ARG, "w4_linear: %zu bytes of workspace, 16-byte aligned, are wanted", wanted);
    // eight values of x at a time where every row allows it
    const size_t vector = 8 * dtype_size(a->dtype), piece = std::min<size_t>(vector, 16);
    const int vectors = reinterpret_cast<uintptr_t>(a->x) % piece == 0 && (a->rows == 1 || a->x_stride * dtype_size(a->dtype) % piece == 0);
    const W4Params p = {static_cast<const uint8_t *>(w->packed), a->x, a->y, a->x_scale, a->bias, a->x_stride, a->y_stride, static_cast<long long>(l.unit_bytes),
                        l.n, l.k, l.tiles, l.units, a->rows, a->dtype, l.wide, l.spans, vectors, a->out_dtype, 0, 0, 0, 0, 0, 0, wanted ? static_cast<uint8_t *>(a->workspace) : nullptr, nullptr, ctx->dev_err_flag, 0};
    if (const int rc = check_device_flag(ctx, ctx->err_flag)) return rc;        // (a call before this one)
    const cudaError_t e = a->dtype == MSNH_B200_F32  ? launch<float>(ctx, p, stream)
                        : a->dtype == MSNH_B200_F16  ? launch<__half>(ctx, p, stream)
                        : a->dtype == MSNH_B200_BF16 ? launch<__nv_bfloat16>(ctx, p, stream)
                                                     : launch<__nv_fp8_e4m3>(ctx, p, stream);
    CUDA_TRY(ctx, e);
    return MSNH_B200_OK;
} catch (...) { return caught(ctx); }

}  // extern "C"
