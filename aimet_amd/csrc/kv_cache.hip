// A key/value cache held in 8 bits, and the attention that reads it.
//
// Stored: codes in [-127, 127], as bytes code + 128, and for every block of `block` tokens (16, 32 or 64) of a sequence and
// head the largest magnitude `amax` among them; a code stands for code * amax / 127.  Both lie as [sequence, head, tile of
// 64 tokens], and inside a tile in pieces of 1 KB that one load of a wave takes whole, 16 bytes a lane, in the order of the
// operands of a 16 x 16 x 32 matrix instruction (key_offset, value_offset): lane 16 c + i of a keys' piece holds 16 channels
// of one token, of a values' piece 16 tokens of one channel.
//
// Writing (kv_append_kernel): a workgroup owns one block of one head.  amax = max(what the block had, |new tokens|), code =
// rint(127 x / amax), half to even and exact; where amax grows, the codes the block had become rint(code * old / new).
//
// Reading (kv_attend_kernel): one pass over the tokens with a running reference and sum of the softmax.  Rows are the query
// heads of one key head, query after query.  A wave takes 64 tokens at a time: scores = keys (A) x queries (B) on the
// matrix cores, so that lane 16 c + i of the result holds 16 tokens of row i.  Keys are handed to the instruction in an
// order that makes those the tokens 16 c .. 16 c + 15 of the tile: that is the B operand of the next product, values (A) x
// probabilities (B), without any exchange between lanes.
//
// Both products run in float16 with float32 sums.  Codes are exact in it: a byte b next to the byte 0x64 is the number
// 1024 + b, and one packed addition of -1152 makes two codes of two bytes.  A query row is multiplied by the power of two
// that brings its largest value to 2^13 .. 2^14 (float16 rows that are larger stay as they are), which keeps 16-bit
// queries exact (bfloat16 down to 2^-30 of the row's largest value); float32 queries become two parts, 22 bits.
// Probabilities carry the scale of their values' block: with x = score + log2(scale), weights are 2^(x - reference), the
// reference being such that the largest weight so far lies between 2^10 and 2^15 (it is moved, and the sums with it, only
// when a weight passes 2^15).  Weights are two float16 parts for queries of every type: off by at most 2^-22 of themselves,
// and by 2^-25 where they are small, 2^-35 of the largest.
// One part (2^-11) would show in 16-bit answers: those of decoding then differ from a float32 softmax's by 4e-4 relative,
// with two by 3e-5 or not at all, at the same time; prompts pay for it (2048 of 3048 tokens: 147 -> 192 us).  The softmax's
// denominator sums weight / scale in float32.  Scales are counted in a unit of the workgroup's share, a power of two: 1 where
// the largest maximum in it is between 2^-5 and 2^16, and otherwise that maximum's, so that values of any size have the same
// precision.  Scales below 2^-84 of the unit count as that, which is what blocks of zeros weigh their tokens with.

#include "../../include/aimet_amd_serving.h"
#include "ahq_host.h"
#include "mma.h"

namespace ahq {

constexpr int kKvTile = 64;
constexpr int kCodeBias = 128;

// Place of a code in its tile of 64 tokens.  Keys: piece (s, u) holds the channels 64 u .. of the tokens 16 g + 4 s + r, lane
// 16 c + 4 g + r those from 64 u + 16 c on.  Values: piece u holds the channels 16 u + i, lane 16 c + i the tokens from
// 16 c on.
template <int D>
__device__ __forceinline__ int key_offset(int token, int channel) {
    const int s = token >> 2 & 3, i = (token >> 4) * 4 + (token & 3);
    return (((s * (D / 64) + (channel >> 6)) * 4 + (channel >> 4 & 3)) * 16 + i) * 16 + (channel & 15);
}
__device__ __forceinline__ int value_offset(int token, int channel) {
    return (((channel >> 4) * 4 + (token >> 4)) * 16 + (channel & 15)) * 16 + (token & 15);
}

// ------------------------------------------------------------------------------------------------------------ append --
struct KvAppendArgs {
    const void* x[2];        // new keys, new values
    int64_t sb[2], sh[2], st[2];  // strides in elements: sequence, head, token
    uint8_t* codes[2];
    float* amax[2];
    const int32_t* start;    // null: start0 for every sequence
    const int32_t* counts;   // null: count0
    int32_t start0, count0;
    int32_t heads, tokens, capacity;
    int32_t vec;             // rows of x start on 16-byte boundaries
};

struct TokenRange { int begin, end; };
// Positions [begin, end) of sequence b that this call writes, and `begin` of the first token of x (may be negative: such
// tokens are not written, nor are those at or behind the capacity).
__device__ __forceinline__ TokenRange new_tokens(const int32_t* start, int start0, const int32_t* counts, int count0,
                                                 int tokens, int capacity, int b) {
    const int s = start ? start[b] : start0;
    int n = counts ? counts[b] : count0;
    n = n < 0 ? 0 : n > tokens ? tokens : n;
    int64_t e = (int64_t)s + n;
    if (e > capacity) e = capacity;
    if (e < 0) e = 0;
    return {s, (int)e};
}

__device__ __forceinline__ float finite_magnitude(float v) {
    const float m = fabsf(v);
    return m < __builtin_inff() ? m : 0.0f;  // neither infinities nor NaN set a block's scale
}

// rint(127 v / amax) + 128, half to even and exact, as the low byte of the result.
//
// Fast form, for finite values of at most 11 bits under a maximum of as many: 127 v is exact (18 bits), and the quotient's
// first estimate, corrected once with its exact remainder, is the rounded quotient.  One that lies half-way between two
// codes has few bits and is met exactly; any other between 2^(6-j) and 2^(7-j) is at least 2^-(12+j) away from half-way,
// 64 times its rounding error.  Adding 1.5 * 2^23 + 128 rounds to a whole number, half to even, and leaves it in the low bits.
__device__ __forceinline__ uint32_t to_byte_fast(float v, float amax, float inverse) {
    const float t = 127.0f * v;
    const float q = t * inverse;
    const float q1 = __builtin_fmaf(__builtin_fmaf(-q, amax, t), inverse, q);
    return f32_to_bits(q1 + 12583040.0f);
}
// Every other case: the remainder of the float64 estimate is exact (31 and 31 bits) and says which neighbour is nearer.
__device__ __forceinline__ uint32_t to_byte_exact(float v, float amax, double inverse) {
    if (v != v) return kCodeBias;
    const double w = fmin(fmax((double)v, -(double)amax), (double)amax);
    double q = __builtin_rint(w * inverse);
    const double twice = 2.0 * __builtin_fma(-q, (double)amax, 127.0 * w);
    const bool odd = ((int)q & 1) != 0;
    if (twice > amax || (odd && twice == amax)) q += 1.0;
    if (twice < -amax || (odd && twice == -amax)) q -= 1.0;
    return (uint32_t)((int)q + kCodeBias);
}
__device__ __forceinline__ uint32_t pack_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return hi << 16 | lo;
}

// A thread has four tokens and eight channels of the block.  Bound by the memory traffic of long prompts, by the launch
// for single tokens: the block is read once, its maximum found with integer comparisons (a pair of 16-bit values at a
// time), and its codes go through LDS so that whole runs of the tile's order are written, without bank conflicts.
// 2047 tokens of 4 x 8 x 128 bfloat16 (50 MB): 13.7 us, 3.7 TB/s; three tokens of 16 x 32 x 64 float16: 4.6 us.
template <int D, int BT> constexpr int kAppendItems = BT / 4 * (D / 8);
template <int D, int BT> constexpr int kAppendThreads = kAppendItems<D, BT> < kWave ? kWave : kAppendItems<D, BT>;

template <typename T, int D, int BT>
__global__ __launch_bounds__((kAppendThreads<D, BT>)) void kv_append_kernel(KvAppendArgs a) {
    constexpr int kThreads = kAppendThreads<D, BT>;
    constexpr int kPairs = sizeof(T) == 2 ? 4 : 8;  // registers of eight values
    const int which = blockIdx.z;
    const int bh = blockIdx.y, b = bh / a.heads, h = bh % a.heads;
    const TokenRange range = new_tokens(a.start, a.start0, a.counts, a.count0, a.tokens, a.capacity, b);
    const int lo = range.begin < 0 ? 0 : range.begin;
    if (lo >= range.end) return;
    const int blk = lo / BT + blockIdx.x;
    const int p0 = blk * BT;
    if (p0 >= range.end) return;
    const int old_end = lo > p0 ? lo - p0 : 0;                       // tokens of the block that were there before
    const int new_end = range.end - p0 < BT ? range.end - p0 : BT;   // [old_end, new_end) are written

    float* amax_at = a.amax[which] + (int64_t)bh * (a.capacity / BT) + blk;
    const float before = old_end > 0 ? *amax_at : 0.0f;
    const T* x = static_cast<const T*>(a.x[which]) + b * a.sb[which] + h * a.sh[which];
    const bool item = kAppendItems<D, BT> >= kWave || threadIdx.x < kAppendItems<D, BT>;
    const int quad = threadIdx.x / (D / 8), d = threadIdx.x % (D / 8) * 8;
    uint32_t raw[4][kPairs];
    const auto value = [&](int r, int e) {
        if constexpr (sizeof(T) == 4) return bits_to_f32(raw[r][e]);
        else return load_f32(T{(uint16_t)(raw[r][e / 2] >> (16 * (e & 1)))});
    };
    uint32_t top = 0;  // of the magnitudes' bit patterns, which are ordered as the magnitudes are
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int t = 4 * quad + r;
#pragma unroll
        for (int e = 0; e < kPairs; ++e) raw[r][e] = 0;
        if (item && t >= old_end && t < new_end) {
            const T* row = x + (int64_t)(p0 + t - range.begin) * a.st[which] + d;
            if (a.vec) {
#pragma unroll
                for (int u = 0; u < kPairs / 4; ++u) {
                    const u32x4_t w = reinterpret_cast<const u32x4_t*>(row)[u];
#pragma unroll
                    for (int e = 0; e < 4; ++e) raw[r][4 * u + e] = w[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (sizeof(T) == 4) raw[r][e] = f32_to_bits(row[e]);
                    else raw[r][e / 2] |= (uint32_t)row[e].bits << (16 * (e & 1));
                }
            }
        }
#pragma unroll
        for (int e = 0; e < kPairs; ++e) {
            if constexpr (sizeof(T) == 4) {
                const uint32_t m = raw[r][e] & 0x7fffffffu;
                top = m > top ? m : top;
            } else {
                typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
                top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                                             __builtin_bit_cast(u16x2, raw[r][e] & 0x7fff7fffu)));
            }
        }
    }
    __shared__ float part[kThreads / kWave];
    const auto over_block = [&](float v) {
        v = wave_reduce(v, OpMaxF());
        if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / kWave; ++w) v = fmaxf(v, part[w]);
        return v;
    };
    float size;
    if constexpr (sizeof(T) == 4) size = bits_to_f32(top);
    else size = load_f32(T{(uint16_t)((top & 0xffffu) > (top >> 16) ? top & 0xffffu : top >> 16)});
    // NaN loses every comparison: it goes through the maximum as an infinity
    float most = over_block(size == size ? size : __builtin_inff());
    const bool special = !(most < __builtin_inff());  // the same for the whole workgroup
    if (special) {
        float finite = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) finite = fmaxf(finite, finite_magnitude(value(r, e)));
        __syncthreads();
        most = over_block(finite);
    }
    const float amax = fmaxf(before, most);
    const bool rescale = old_end > 0 && amax > before;
    const int first = rescale ? 0 : old_end;  // first token whose codes are stored

    uint8_t* tile = a.codes[which] + ((int64_t)bh * a.capacity + p0 / kKvTile * kKvTile) * D;
    const int t0 = p0 % kKvTile;  // the block's first token in its tile
    uint32_t code[4][8];
    if (!(amax > 0.0f)) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) code[r][e] = kCodeBias;
    } else if (sizeof(T) == 2 && !special && amax > 1e-30f && amax < 1e36f && (f32_to_bits(amax) & 0x1fffu) == 0) {
        const float inverse = 1.0f / amax;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) code[r][e] = to_byte_fast(value(r, e), amax, inverse);
    } else {
        const double inverse = 127.0 / (double)amax;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) code[r][e] = to_byte_exact(value(r, e), amax, inverse);
    }
    if (rescale && item && 4 * quad < old_end) {
        for (int r = 0; r < 4; ++r) {
            const int t = 4 * quad + r;
            if (t >= old_end) break;
            for (int e = 0; e < 8; ++e) {
                const int q = tile[which ? value_offset(t0 + t, d + e) : key_offset<D>(t0 + t, d + e)] - kCodeBias;
                const uint32_t v = (uint32_t)((int)__builtin_rint((double)q * (double)before / (double)amax) + kCodeBias);
#pragma unroll
                for (int rr = 0; rr < 4; ++rr)
#pragma unroll
                    for (int ee = 0; ee < 8; ++ee) code[rr][ee] = rr == r && ee == e ? v : code[rr][ee];
            }
        }
    }
    constexpr int kRun = BT / 4 * 16, kPitch = D + 4;  // bytes of a run of the keys' order; channels of a row of quads
    __shared__ alignas(16) uint8_t stage[D / 4 * (kRun + 16) > BT * kPitch ? D / 4 * (kRun + 16) : BT * kPitch];
    if (which == 0) {
        if (item) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                u32x2_t w = {pack_bytes(code[r][0], code[r][1], code[r][2], code[r][3]), pack_bytes(code[r][4], code[r][5], code[r][6], code[r][7])};
                *reinterpret_cast<u32x2_t*>(stage + ((quad & 3) * (D / 16) + d / 16) * (kRun + 16) + ((quad >> 2) * 4 + r) * 16 + (d & 8)) = w;
            }
        }
        __syncthreads();
        for (int id = threadIdx.x; id < BT * D / 16; id += kThreads) {
            const int i = id % (BT / 4), run = id / (BT / 4);
            const int t = (i >> 2) * 16 + run / (D / 16) * 4 + (i & 3);
            if (t >= first && t < new_end)
                *reinterpret_cast<u32x4_t*>(tile + run * 256 + (t0 / 4 + i) * 16) = *reinterpret_cast<const u32x4_t*>(stage + run * (kRun + 16) + i * 16);
        }
    } else {
        uint32_t* quads = reinterpret_cast<uint32_t*>(stage);  // four tokens of a channel: [quad][channel]
        if (item) {
            u32x4_t w[2];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e / 4][e % 4] = pack_bytes(code[0][e], code[1][e], code[2][e], code[3][e]);
            *reinterpret_cast<u32x4_t*>(quads + quad * kPitch + d) = w[0];
            *reinterpret_cast<u32x4_t*>(quads + quad * kPitch + d + 4) = w[1];
        }
        __syncthreads();
        for (int id = threadIdx.x; id < BT * D / 16; id += kThreads) {
            const int i = id & 15, c = (id >> 4) % (BT / 16), u = (id >> 4) / (BT / 16);
            u32x4_t w;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = quads[(4 * c + j) * kPitch + 16 * u + i];
            uint8_t* to = tile + (u * 4 + t0 / 16 + c) * 256 + i * 16;
            const int t = 16 * c;
            if (first <= t && t + 16 <= new_end) {
                *reinterpret_cast<u32x4_t*>(to) = w;
            } else {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (t + e >= first && t + e < new_end) to[e] = (uint8_t)(w[e / 4] >> (8 * (e & 3)));
            }
        }
    }
    // read by all threads before the first barrier above, so it is written behind one
    if (threadIdx.x == 0) *amax_at = amax;
}

// -------------------------------------------------------------------------------------------------------- dequantize --
struct KvValuesArgs {
    const uint8_t* codes[2];
    const float* amax[2];
    void* out[2];  // [sequence, head, length, D]
    int32_t capacity, length, block_shift;
};

// A workgroup has one tile of 64 tokens.  Bound by memory: the tile is read whole and in order, and turned round in LDS
// (keys: runs of 256 bytes 16 apart; values: [four tokens][channel + 4]), both without bank conflicts.  303 tokens of
// 16 x 32 x 64 to float16 (60 MB): 10.1 us, 5.9 TB/s.
template <typename T, int D>
__global__ __launch_bounds__(kBlock) void kv_values_kernel(KvValuesArgs a) {
    constexpr int kPitch = D + 4;
    const int which = blockIdx.z, tile = blockIdx.x;
    const int64_t bh = blockIdx.y;
    const int p0 = tile * kKvTile;
    const u32x4_t* codes = reinterpret_cast<const u32x4_t*>(a.codes[which] + (bh * a.capacity + p0) * D);
    const float* amax = a.amax[which] + (bh * a.capacity >> a.block_shift);
    T* out = static_cast<T*>(a.out[which]) + (bh * a.length + p0) * D;
    static_assert(68 * D >= 64 * kPitch, "the keys' image is the larger");
    __shared__ alignas(16) uint8_t stage[68 * D];
    uint32_t* quads = reinterpret_cast<uint32_t*>(stage);
    for (int id = threadIdx.x; id < D * 4; id += kBlock) {
        const u32x4_t w = codes[id];
        if (which == 0) {
            *reinterpret_cast<u32x4_t*>(stage + id * 16 + (id >> 4) * 16) = w;
        } else {
            const int i = id & 15, c = id >> 4 & 3, u = id >> 6;
#pragma unroll
            for (int j = 0; j < 4; ++j) quads[(4 * c + j) * kPitch + 16 * u + i] = w[j];
        }
    }
    __syncthreads();
    const auto store = [&](int t, int d, const float* v) {  // eight channels of a token
        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
        for (int u = 0; u < 8 / kPer; ++u) {
            Pack<T, kPer> w;
#pragma unroll
            for (int e = 0; e < kPer; ++e) w.v[e] = store_cast<T>(v[u * kPer + e]);
            store_pack<T, kPer>(out + (int64_t)t * D + d + u * kPer, w);
        }
    };
    // The code is exact, so its product with the scale is rounded once.  float16: as (byte - 128) * scale in one instruction
    // with the rounding to float16; larger scales than 2^100 make infinities of all codes but 0 either way.  float32: the
    // scale of the largest number is rounded up, and 127 times that would be infinite.
    const auto scaled = [](uint32_t w, int byte, float s) {
        if constexpr (sizeof(T) == 4)
            return __builtin_amdgcn_fmed3f((float)(int8_t)((w ^ 0x80808080u) >> (8 * byte)) * s, -3.402823466e38f, 3.402823466e38f);
        else if constexpr (std::is_same_v<T, f16_t>)
            return __builtin_fmaf((float)(w >> (8 * byte) & 0xffu), s, -128.0f * s);
        else
            return (float)(int8_t)((w ^ 0x80808080u) >> (8 * byte)) * s;
    };
    for (int id = threadIdx.x; id < 16 * (D / 8); id += kBlock) {
        const int quad = id / (D / 8), d = id % (D / 8) * 8;
        if (p0 + 4 * quad >= a.length) break;
        float s = amax[(p0 + 4 * quad) >> a.block_shift] / 127.0f;
        if constexpr (std::is_same_v<T, f16_t>) s = fminf(s, 0x1p100f);
        u32x4_t w[2];
        if (which) {
            w[0] = *reinterpret_cast<const u32x4_t*>(quads + quad * kPitch + d);
            w[1] = *reinterpret_cast<const u32x4_t*>(quads + quad * kPitch + d + 4);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = 4 * quad + r;
            float v[8];
            if (which) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = scaled(w[e / 4][e % 4], r, s);
            } else {
                const int at = key_offset<D>(t, d);
                const u32x2_t k = *reinterpret_cast<const u32x2_t*>(stage + at + (at >> 8) * 16);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = scaled(k[e / 4], e % 4, s);
            }
            if (p0 + t < a.length) store(t, d, v);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ attend --
struct KvAttendArgs {
    const void* q;
    void* out;
    int64_t qb, qh, qt, ob, oh, ot;  // strides in elements
    const uint8_t *k_codes, *v_codes;
    const float *k_amax, *v_amax;
    const int32_t* lengths;  // null: length0
    const int32_t* counts;   // null: count0
    int32_t length0, count0;
    int32_t heads, groups, queries, capacity, block_shift;
    int32_t rows, row_tile;       // queries * groups; rows of a workgroup
    int32_t splits, split_tiles;  // splits of the token axis, token tiles of each
    float scale;                  // of the scores, times log2(e)
    int32_t vec;                  // rows of q start on 16-byte boundaries
    int32_t vec_out;              // rows of the answers start on boundaries of four elements
    float* part;                  // [sequence * head][row][split][D], then [..][row][split][2]: reference and sum
    float* part_stat;
};

struct SequenceView { int length, count; };
__device__ __forceinline__ SequenceView view_sequence(const KvAttendArgs& a, int b) {
    int n = a.lengths ? a.lengths[b] : a.length0;
    int t = a.counts ? a.counts[b] : a.count0;
    n = n < 0 ? 0 : n > a.capacity ? a.capacity : n;
    t = t < 0 ? 0 : t > a.queries ? a.queries : t;
    return {n, t};
}
// Token tiles that hold something the rows up to `row` see.
__device__ __forceinline__ int seen_tiles(const KvAttendArgs& a, const SequenceView& seq, int row) {
    int t = row / a.groups;
    if (t >= seq.count) t = seq.count - 1;
    const int seen = seq.length - seq.count + t + 1;
    return t < 0 || seen <= 0 ? 0 : (seen + kKvTile - 1) / kKvTile;
}
// Largest of the lane's part of the blocks' maxima that a share's rows up to `row` see: those of its tiles [first, stop).
// Blocks behind the last token hold the scales of other ones.
__device__ __forceinline__ float seen_amax(const KvAttendArgs& a, const SequenceView& seq, const float* amax, int row, int first, int stop) {
    int t = row / a.groups;
    if (t >= seq.count) t = seq.count - 1;
    const int tokens = seq.length - seq.count + t + 1, until = stop * kKvTile < tokens ? stop * kKvTile : tokens;
    const int last = until > 0 ? (until - 1) >> a.block_shift : 0;
    int at = (first * kKvTile >> a.block_shift) + (int)(threadIdx.x & (kWave - 1));
    float most = amax[at < last ? at : last];  // not a masked load: short shares have no more than this one
    for (at += kWave; at <= last; at += kWave) most = fmaxf(most, amax[at]);
    return most;
}
// Splits of the token axis that hold such tiles, for the workgroup's rows that `row` is one of.
__device__ __forceinline__ int used_splits(const KvAttendArgs& a, const SequenceView& seq, int row) {
    return (seen_tiles(a, seq, row / a.row_tile * a.row_tile + a.row_tile - 1) + a.split_tiles - 1) / a.split_tiles;
}

// Two codes of the low or of the high half of a word, exact in float16.
__device__ __forceinline__ f16x2 two_codes(uint32_t w, uint32_t selector) {
    const f16x2 biased = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, selector));
    return biased + f16x2{(_Float16)-1152.0f, (_Float16)-1152.0f};
}
__device__ __forceinline__ f16x8 codes_to_f16(uint32_t a, uint32_t b) {
    union { f16x2 h[4]; f16x8 v; } r;
    r.h[0] = two_codes(a, 0x04010400u), r.h[1] = two_codes(a, 0x04030402u);
    r.h[2] = two_codes(b, 0x04010400u), r.h[3] = two_codes(b, 0x04030402u);
    return r.v;
}
__device__ __forceinline__ f16x8 half_piece(const u32x4_t& w, int half) { return codes_to_f16(w[2 * half], w[2 * half + 1]); }
// Eight values as a sum of N float16 fragments.
template <int N>
__device__ __forceinline__ void split_f16(const float* v, f16x8* out) {
    float rest[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) rest[e] = v[e];
#pragma unroll
    for (int p = 0; p < N; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            out[p][e] = (_Float16)rest[e];
            if (p + 1 < N) rest[e] = __builtin_fmaf((float)out[p][e], -1.0f, rest[e]);
        }
}

// Largest value over the four lanes of a row, which are 16 apart.
__device__ __forceinline__ float row_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(f32_to_bits(v), f32_to_bits(v), false, false);
    v = fmaxf(bits_to_f32(a[0]), bits_to_f32(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(f32_to_bits(v), f32_to_bits(v), false, false);
    return fmaxf(bits_to_f32(b[0]), bits_to_f32(b[1]));
}

// An answer is an average of finite values: it is no larger than they are, whatever its roundings.  NaN stays.
__device__ __forceinline__ float finite(float v) {
    return v > 3.402823466e38f ? 3.402823466e38f : v < -3.402823466e38f ? -3.402823466e38f : v;
}

constexpr float kTop = 15.0f, kStart = 10.0f;  // log2 of the largest weight: at most, and where the reference is set to
constexpr float kLeastScale = 0x1p-84f;  // in units
constexpr float kOrdinary = 0x1p-5f, kLarge = 0x1p16f;  // maxima that are counted in the unit 1
constexpr int kLeastUnit = -126, kLargestUnit = 118;    // 2^-unit / 127 is a normal number
constexpr int kAttendWaves = 4;

// What a wave knows of its 16 * NR rows; a lane holds row 16 n + i of them and the channels 16 u + 4 c + r of its answer.
template <typename T, int D, int NR>
struct AttendRows {
    static constexpr int kParts = sizeof(T) == 4 ? 2 : 1;
    static constexpr int kSteps = D / 32, kOut = D / 16;
    static constexpr int kWeightParts = 2;  // of the probabilities, for every type
    f16x8 q[kSteps][NR][kParts];
    f32x4 o[kOut][NR];
    float rescale[NR];  // what the row's power of two is undone with, times the scale of the scores
    float reference[NR], top[NR], sum[NR];
    int last[NR];       // the last token the row sees; below 0: none
    int least;          // of the wave's rows that see anything, the least `last`
    int unit;           // scales of values are counted in 2^unit
    float to_unit;      // 2^-unit / 127

    __device__ __forceinline__ void begin(const KvAttendArgs& a, const SequenceView& seq, int b, int h, int row0, int i, int c) {
        least = 0x7fffffff;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int row = row0 + 16 * n + i, t = row / a.groups;
            last[n] = row < a.rows && t < seq.count ? seq.length - seq.count + t : -1;
            const bool live = last[n] >= 0;
            if (live && last[n] < least) least = last[n];
            // rows that see nothing read the first query's place and count as zero
            const T* at = static_cast<const T*>(a.q) + b * a.qb + (int64_t)(h * a.groups + (live ? row % a.groups : 0)) * a.qh + (int64_t)(live ? t : 0) * a.qt + 16 * c;
            float v[kSteps][8];
            if (a.vec) {
                constexpr int kPer = 16 / sizeof(T);
                Pack<T, kPer> raw[kSteps][8 / kPer];
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int u = 0; u < 8 / kPer; ++u) raw[s][u] = load_pack<T, kPer>(at + 64 * (s / 2) + 8 * (s % 2) + u * kPer);
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[s][e] = load_f32(raw[s][e / kPer].v[e % kPer]);
            } else {
#pragma unroll
                for (int s = 0; s < kSteps; ++s)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[s][e] = load_f32(at[64 * (s / 2) + 8 * (s % 2) + e]);
            }
            float size = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[s][e] = live ? v[s][e] : 0.0f;
                    size = fmaxf(size, fabsf(v[s][e]));
                }
            size = row_max(size);
            // exponent of the largest value; zeros, infinities and the smallest numbers go as they are
            int ex = (int)(f32_to_bits(size) >> 23);
            if (size == 0.0f || ex >= 255) ex = 140;
            if (ex < 16) ex = 16;
            // float16 is never scaled down: its smallest numbers would lose bits, and its largest fit as they are
            if (std::is_same_v<T, f16_t> && ex > 140) ex = 140;
            const float up = bits_to_f32((uint32_t)(267 - ex) << 23);
            rescale[n] = bits_to_f32((uint32_t)(ex - 13) << 23) * a.scale;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[s][e] *= up;
                split_f16<kParts>(v[s], q[s][n]);
            }
            reference[n] = 0.0f, top[n] = -__builtin_inff(), sum[n] = 0.0f;
#pragma unroll
            for (int u = 0; u < kOut; ++u) o[u][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int m = 1; m < 16; m *= 2) {
            const int other = __shfl_xor(least, m, kWave);
            least = other < least ? other : least;
        }
        least = __builtin_amdgcn_readfirstlane(least);
    }
    // The unit, from the largest of the lanes' maxima; a share of zeros has any.
    __device__ __forceinline__ void set_unit(float most) {
        unit = 0;
        if (__builtin_expect(__any(most >= kLarge) || !__any(most >= kOrdinary), 0)) {
            most = wave_reduce(most, OpMaxF());
            const int e = __builtin_amdgcn_readfirstlane((int)(f32_to_bits(most) >> 23) - 127);
            unit = e < kLeastUnit ? kLeastUnit : e > kLargestUnit ? kLargestUnit : e;
        }
        to_unit = bits_to_f32((uint32_t)(127 - unit) << 23) * (1.0f / 127.0f);
    }

    // One tile of 64 tokens from p0 on: `key(s, u)` and `value(u, w)` give operands, `between` is called once the keys and
    // scales are no longer needed.  AHEAD: operands come from LDS and are asked for one group of products early, in an
    // order that the compiler keeps (its own waits for each one right behind its load).
    template <bool AHEAD, typename Key, typename Value, typename Between>
    __device__ __forceinline__ void work(Key key, Value value, float k_amax, float v_amax, int p0, int c, Between between) {
        const float k_scale = k_amax * (1.0f / 127.0f);
        const float v_scale = fmaxf(v_amax * to_unit, kLeastScale);
        const float v_log = __builtin_amdgcn_logf(v_scale);
        const float v_inverse = __builtin_amdgcn_rcpf(v_scale);
        f32x4 x[4][NR];
        f16x8 kf[2][kSteps];
#pragma unroll
        for (int u = 0; u < kSteps; ++u) kf[0][u] = key(0, u);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (s < 3) {
#pragma unroll
                for (int u = 0; u < kSteps; ++u) kf[(s + 1) % 2][u] = key(s + 1, u);
            }
            if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < NR; ++n) x[s][n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < kSteps; ++u)
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int p = 0; p < kParts; ++p) x[s][n] = mma(kf[s % 2][u], q[u][n][p], x[s][n]);
            if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
        }
        between();
        f16x8 vf[3][2];
        if constexpr (AHEAD) {
#pragma unroll
            for (int u = 0; u < 2; ++u) vf[u][0] = value(u, 0), vf[u][1] = value(u, 1);
        }
        f16x8 pf[2][NR][kWeightParts];
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const float factor = k_scale * rescale[n], shift = v_log - reference[n];
            float most = -__builtin_inff();
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) x[s][n][r] = __builtin_fmaf(x[s][n][r], factor, shift);
            float inverse = v_inverse;
            if (p0 + kKvTile - 1 > least) {  // some row's last token lies in this tile
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (p0 + 16 * c + 4 * s + r > last[n]) x[s][n][r] = -__builtin_inff();
                if (p0 + 16 * c > last[n]) inverse = 0.0f;
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) most = fmaxf(most, x[s][n][r]);
            most = row_max(most);
            const bool raise = most > top[n];
            if (__any(raise)) {  // seldom once a few tiles are done
                const float by = raise ? most - kStart : 0.0f;
                const float fade = !raise ? 1.0f : top[n] == kTop ? __builtin_amdgcn_exp2f(-by) : 0.0f;
                if (raise) top[n] = kTop;
                reference[n] += by;
                sum[n] *= fade;
#pragma unroll
                for (int u = 0; u < kOut; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[u][n][r] *= fade;
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[s][n][r] -= by;
            }
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    p[e] = __builtin_amdgcn_exp2f(x[2 * w + e / 4][n][e % 4]);
                    total += p[e];
                }
                split_f16<kWeightParts>(p, pf[w][n]);
            }
            sum[n] = __builtin_fmaf(total, inverse, sum[n]);
        }
#pragma unroll
        for (int u = 0; u < kOut; ++u) {
            if constexpr (AHEAD) {
                if (u + 2 < kOut) vf[(u + 2) % 3][0] = value(u + 2, 0), vf[(u + 2) % 3][1] = value(u + 2, 1);
                __builtin_amdgcn_sched_barrier(0);
            } else {
                vf[u % 3][0] = value(u, 0), vf[u % 3][1] = value(u, 1);
            }
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int p = 0; p < kWeightParts; ++p) {
                    o[u][n] = mma(vf[u % 3][0], pf[0][n][p], o[u][n]);
                    o[u][n] = mma(vf[u % 3][1], pf[1][n][p], o[u][n]);
                }
        }
    }
};

// The rows' answers, or their share of them where the token axis is split: from a wave's registers.
template <typename T, int D, int NR>
__device__ __forceinline__ void store_rows(const KvAttendArgs& a, const AttendRows<T, D, NR>& rows, const float* sum, int64_t bh,
                                           int row0, int split, bool whole, int i, int c) {
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        const int row = row0 + 16 * n + i;
        if (row >= a.rows) continue;
        if (whole) {
            const float inverse = sum[n] == 0.0f ? 0.0f : 1.0f / sum[n];
            T* to = static_cast<T*>(a.out) + b * a.ob + (int64_t)(h * a.groups + row % a.groups) * a.oh + (int64_t)(row / a.groups) * a.ot + 4 * c;
#pragma unroll
            for (int u = 0; u < D / 16; ++u) {
                Pack<T, 4> out;
#pragma unroll
                for (int r = 0; r < 4; ++r) out.v[r] = store_cast<T>(sum[n] == 0.0f ? 0.0f : finite(rows.o[u][n][r] * inverse));
                if (a.vec_out) {
                    store_pack<T, 4>(to + 16 * u, out);
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r) to[16 * u + r] = out.v[r];
                }
            }
        } else {
            const int64_t at = (bh * a.rows + row) * a.splits + split;
#pragma unroll
            for (int u = 0; u < D / 16; ++u) *reinterpret_cast<f32x4*>(a.part + at * D + 16 * u + 4 * c) = rows.o[u][n];
            if (c == 0) a.part_stat[at * 2] = rows.reference[n], a.part_stat[at * 2 + 1] = sum[n];
        }
    }
}

// Sums over the lanes of a row, in the unit 1; rows that saw nothing have the reference -infinity and the sum 0.  Far units
// are shared out between a row's answer and its sum, so that neither leaves float32; where blocks of zeros have the row's
// weight, the sum is large, and its answer takes the rest.
template <typename T, int D, int NR>
__device__ __forceinline__ void finish_rows(AttendRows<T, D, NR>& rows, float* sum) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        sum[n] = rows.sum[n];
        sum[n] += __shfl_xor(sum[n], 16, kWave);
        sum[n] += __shfl_xor(sum[n], 32, kWave);
        if (__builtin_expect(rows.unit != 0, 0)) {
            int share = rows.unit >= -24 && rows.unit <= 24 ? 0 : rows.unit / 2;
            const int most = 227 + rows.unit - (int)(f32_to_bits(sum[n]) >> 23);  // leaves the sum at 2^101
            if (most < share) share = most;
            if (__any(share != 0)) {
#pragma unroll
                for (int u = 0; u < D / 16; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) rows.o[u][n][r] = __builtin_amdgcn_ldexpf(rows.o[u][n][r], share);
            }
            rows.reference[n] += (float)(rows.unit - share);
            sum[n] = __builtin_amdgcn_ldexpf(sum[n], share - rows.unit);
        }
        if (rows.last[n] < 0) sum[n] = 0.0f;
        if (rows.top[n] != kTop) rows.reference[n] = -__builtin_inff();
    }
}

// Few rows, long caches (decoding): the four waves of a workgroup share its 16 rows and take their token tiles in turn.
// Bound by the stream of codes: keys of the next tile and values of this one are asked for before the work on this one
// begins.  STREAM: the codes are more than the caches keep, so they are read past them.
//
// 131071 tokens of 8 x 128 (268 MB): 50 us, 5.4 TB/s, and 4.6 us for the join; 32 sequences of up to 4096 tokens, 8 x 128
// (134 MB): 35 us in all; 100 tokens of 32 x 64: 4.3 us.
template <typename T, int D, bool STREAM>
__global__ __launch_bounds__(kAttendWaves * kWave, D <= 128 ? 2 : 1) void kv_attend_kernel(KvAttendArgs a) {
    constexpr int kOut = D / 16;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int i = lane & 15, c = lane >> 4;
    const int64_t bh = blockIdx.x;
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
    const int split = blockIdx.z, row0 = (int)(gridDim.y - 1 - blockIdx.y) * 16;  // the rows that see most come first
    const SequenceView seq = view_sequence(a, b);
    const int used = used_splits(a, seq, row0);
    if (split >= used && split > 0) return;

    const int tiles = seen_tiles(a, seq, row0 + 15);
    const int first = split * a.split_tiles + wave;
    const int stop = (split + 1) * a.split_tiles < tiles ? (split + 1) * a.split_tiles : tiles;
    const uint8_t* keys = a.k_codes + bh * a.capacity * D;
    const uint8_t* values = a.v_codes + bh * a.capacity * D;
    const float* k_amax = a.k_amax + bh * (a.capacity >> a.block_shift);
    const float* v_amax = a.v_amax + bh * (a.capacity >> a.block_shift);
    const int amax_at = 16 * c >> a.block_shift;

    // Loads are waited for in the order they were asked for, so a tile's scales come in front of its keys.
    u32x4_t kw[4][D / 64];
    float k_next = 0.0f, v_next = 0.0f;
    const auto piece = [&](const uint8_t* from, int n) {
        const u32x4_t* at = reinterpret_cast<const u32x4_t*>(from + (lane * 16 + n * 1024));
        if constexpr (STREAM) return __builtin_nontemporal_load(at);
        else return *at;
    };
    const auto load = [&](int tile) {
        k_next = k_amax[((int64_t)tile * kKvTile >> a.block_shift) + amax_at];
        v_next = v_amax[((int64_t)tile * kKvTile >> a.block_shift) + amax_at];
        const uint8_t* from = keys + (int64_t)tile * (kKvTile * D);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int u = 0; u < D / 64; ++u) kw[s][u] = piece(from, s * (D / 64) + u);
    };
    const float most = seen_amax(a, seq, v_amax, row0 + 15, split * a.split_tiles, stop);
    if (first < stop) load(first);
    AttendRows<T, D, 1> rows;
    rows.begin(a, seq, b, h, row0, i, c);
    rows.set_unit(most);
    for (int tile = first; tile < stop; tile += kAttendWaves) {
        u32x4_t vw[kOut];
        const uint8_t* from = values + (int64_t)tile * (kKvTile * D);
#pragma unroll
        for (int u = 0; u < kOut; ++u) vw[u] = piece(from, u);
        // behind the last tile that one is loaded again: a load that may be left out would have to be waited for at once
        rows.template work<false>([&](int s, int u) { return half_piece(kw[s][u / 2], u % 2); }, [&](int u, int w) { return half_piece(vw[u], w); },
                  k_next, v_next, tile * kKvTile, c, [&] { load(tile + kAttendWaves < stop ? tile + kAttendWaves : tile); });
    }
    float sum[1];
    finish_rows(rows, sum);

    // the waves' results are joined through LDS, in wave order
    constexpr int kPitch = 17;
    extern __shared__ float joined[];  // [wave][D][17], then [wave][16][2]
    float* stats = joined + kAttendWaves * D * kPitch;
#pragma unroll
    for (int u = 0; u < kOut; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) joined[(wave * D + 16 * u + 4 * c + r) * kPitch + i] = rows.o[u][0][r];
    if (c == 0) stats[(wave * 16 + i) * 2] = rows.reference[0], stats[(wave * 16 + i) * 2 + 1] = sum[0];
    __syncthreads();
    for (int id = threadIdx.x; id < 16 * D; id += kAttendWaves * kWave) {
        const int rr = id / D, d = id % D;
        const int row = row0 + rr;
        if (row >= a.rows) break;
        float best = -__builtin_inff();
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w) best = fmaxf(best, stats[(w * 16 + rr) * 2]);
        const float base = best == -__builtin_inff() ? 0.0f : best;
        float total = 0.0f, value = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttendWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(stats[(w * 16 + rr) * 2] - base);
            total += f * stats[(w * 16 + rr) * 2 + 1];
            value += f * joined[(w * D + d) * kPitch + rr];
        }
        if (used <= 1) {
            T* to = static_cast<T*>(a.out) + b * a.ob + (int64_t)(h * a.groups + row % a.groups) * a.oh + (int64_t)(row / a.groups) * a.ot;
            to[d] = store_cast<T>(total == 0.0f ? 0.0f : finite(value / total));
        } else {
            const int64_t at = (bh * a.rows + row) * a.splits + split;
            a.part[at * D + d] = value;
            if (d == 0) a.part_stat[at * 2] = best, a.part_stat[at * 2 + 1] = total;
        }
    }
}

// Many rows (prompts): each wave has 16 * NR rows of its own, and the workgroup takes the token tiles one after the other
// through two LDS buffers, turned into float16 once for all its waves; the next tile is on its way to registers while this
// one is worked on.  Bound by the matrix cores and the vector work between the two products together.  2048 queries of
// 3048 tokens, 2 x 8 x 4 heads of 128: 192 us, 707 TFLOP/s (1060 with the second parts of the weights).
template <typename T, int D, int NR, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, 2) void kv_prompt_kernel(KvAttendArgs a) {
    constexpr int kThreads = WAVES * kWave;
    constexpr int kPieces = D * kKvTile / 16;             // of 16 bytes, of keys and of values each
    constexpr int kPer = 2 * kPieces / kThreads;
    static_assert(2 * kPieces % kThreads == 0, "whole tiles");
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int i = lane & 15, c = lane >> 4;
    const int64_t bh = blockIdx.x;
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
    const int split = blockIdx.z;
    // the rows that see most come first, those of all heads, so that the workgroups that end the call are short ones
    const int wg_row = (int)(gridDim.y - 1 - blockIdx.y) * a.row_tile;
    const SequenceView seq = view_sequence(a, b);
    const int used = used_splits(a, seq, wg_row);
    if (split >= used && split > 0) return;

    const int row0 = wg_row + wave * 16 * NR;
    const int first = split * a.split_tiles;
    const auto limit = [&](int row) {
        const int tiles = seen_tiles(a, seq, row);
        return first + a.split_tiles < tiles ? first + a.split_tiles : tiles;
    };
    const int stop = limit(wg_row + a.row_tile - 1);
    const int mine = row0 < a.rows ? limit(row0 + 16 * NR - 1) : 0;
    const u32x4_t* keys = reinterpret_cast<const u32x4_t*>(a.k_codes + bh * a.capacity * D);
    const u32x4_t* values = reinterpret_cast<const u32x4_t*>(a.v_codes + bh * a.capacity * D);
    const float* k_amax = a.k_amax + bh * (a.capacity >> a.block_shift);
    const float* v_amax = a.v_amax + bh * (a.capacity >> a.block_shift);
    const int amax_at = 16 * c >> a.block_shift;
    extern __shared__ f16x8 buffers[];  // [2][keys, values][piece of 64 lanes][half][64]

    u32x4_t coming[kPer];
    float k_next = 0.0f, v_next = 0.0f;
    const auto load = [&](int tile) {
        k_next = k_amax[((int64_t)tile * kKvTile >> a.block_shift) + amax_at];
        v_next = v_amax[((int64_t)tile * kKvTile >> a.block_shift) + amax_at];
#pragma unroll
        for (int n = 0; n < kPer; ++n) {
            const int at = n * kThreads + threadIdx.x;
            coming[n] = at < kPieces ? keys[(int64_t)tile * kPieces + at] : values[(int64_t)tile * kPieces + at - kPieces];
        }
    };
    const float most = seen_amax(a, seq, v_amax, wg_row + a.row_tile - 1, first, stop);
    if (first < stop) load(first);
    AttendRows<T, D, NR> rows;
    rows.begin(a, seq, b, h, row0, i, c);
    rows.set_unit(most);
    for (int tile = first; tile < stop; ++tile) {
        f16x8* buffer = buffers + (tile & 1) * 4 * kPieces;
        const float k_now = k_next, v_now = v_next;
#pragma unroll
        for (int n = 0; n < kPer; ++n)
#pragma unroll
            for (int half = 0; half < 2; ++half)
                buffer[(n * WAVES + wave) * 2 * kWave + half * kWave + lane] = half_piece(coming[n], half);
        // one barrier a tile: this buffer was last read two tiles ago, in front of the previous barrier
        __syncthreads();
        load(tile + 1 < stop ? tile + 1 : tile);
        if (tile < mine)
            rows.template work<true>([&](int s, int u) { return buffer[(s * (D / 32) + u) * kWave + lane]; },
                      [&](int u, int w) { return buffer[2 * kPieces + (2 * u + w) * kWave + lane]; }, k_now, v_now, tile * kKvTile, c, [] {});
    }
    float sum[NR];
    finish_rows(rows, sum);
    store_rows(a, rows, sum, bh, row0, split, used <= 1, i, c);
}

// One workgroup per row joins the splits: the weights of all of them first, then 1024 / D splits at a time with 16 bytes
// a lane, their sums through LDS in a fixed order.  Rows that one split answered are done already.
constexpr int kJoinThreads = 256;
template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void kv_join_kernel(KvAttendArgs a) {
    constexpr int kLanes = D / 4, kRows = kJoinThreads / kLanes;
    const int row = blockIdx.x;
    const int64_t bh = blockIdx.y;
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
    const SequenceView seq = view_sequence(a, b);
    const int used = used_splits(a, seq, row);
    if (used <= 1) return;
    const int64_t at = (bh * a.rows + row) * a.splits;
    const float* stat = a.part_stat + at * 2;
    const float* part = a.part + at * D;
    __shared__ float smem[kJoinThreads / kWave];
    __shared__ float weight[kJoinThreads];
    __shared__ f32x4 sums[kRows][kLanes];
    float best = -__builtin_inff();
    for (int s = threadIdx.x; s < used; s += kJoinThreads) best = fmaxf(best, stat[(int64_t)s * 2]);
    best = block_reduce(best, OpMaxF(), smem);
    const float base = best == -__builtin_inff() ? 0.0f : best;
    float total = 0.0f;
    f32x4 value = {0.f, 0.f, 0.f, 0.f};
    const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
    for (int s0 = 0; s0 < used; s0 += kJoinThreads) {
        const int s = s0 + threadIdx.x;
        __syncthreads();
        if (s < used) {
            const float f = __builtin_amdgcn_exp2f(stat[(int64_t)s * 2] - base);
            weight[threadIdx.x] = f;
            total += f * stat[(int64_t)s * 2 + 1];
        }
        __syncthreads();
        const int n = used - s0 < kJoinThreads ? used - s0 : kJoinThreads;
#pragma unroll 4
        for (int j = group; j < n; j += kRows) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(part + (int64_t)(s0 + j) * D + 4 * lane);
            const float f = weight[j];
#pragma unroll
            for (int r = 0; r < 4; ++r) value[r] = __builtin_fmaf(f, v[r], value[r]);
        }
    }
    total = block_reduce(total, OpAddF(), smem);
    sums[group][lane] = value;
    __syncthreads();
    if (group) return;
    for (int j = 1; j < kRows; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) value[r] += sums[j][lane][r];
    T* to = static_cast<T*>(a.out) + b * a.ob + (int64_t)(h * a.groups + row % a.groups) * a.oh + (int64_t)(row / a.groups) * a.ot + 4 * lane;
#pragma unroll
    for (int r = 0; r < 4; ++r) to[r] = store_cast<T>(total == 0.0f ? 0.0f : finite(value[r] / total));
}

// The same for up to eight splits, where rows are many: D / 4 lanes to a row (1024 queries of 1 x 8 x 4 heads in two
// splits: 32 us less than with a workgroup for each row).
template <typename T, int D>
__global__ __launch_bounds__(kJoinThreads) void kv_join_rows_kernel(KvAttendArgs a) {
    constexpr int kLanes = D / 4, kRows = kJoinThreads / kLanes;
    const int row = blockIdx.x * kRows + threadIdx.x / kLanes, lane = threadIdx.x % kLanes;
    const int64_t bh = blockIdx.y;
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
    if (row >= a.rows) return;
    const int used = used_splits(a, view_sequence(a, b), row);
    if (used <= 1) return;
    const int64_t at = (bh * a.rows + row) * a.splits;
    const float* stat = a.part_stat + at * 2;
    const f32x4* part = reinterpret_cast<const f32x4*>(a.part + at * D) + lane;
    float best = -__builtin_inff();
    for (int s = 0; s < used; ++s) best = fmaxf(best, stat[2 * s]);
    const float base = best == -__builtin_inff() ? 0.0f : best;
    float total = 0.0f;
    f32x4 value = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < used; ++s) {
        const float f = __builtin_amdgcn_exp2f(stat[2 * s] - base);
        const f32x4 v = part[s * kLanes];
        total = __builtin_fmaf(f, stat[2 * s + 1], total);
#pragma unroll
        for (int r = 0; r < 4; ++r) value[r] = __builtin_fmaf(f, v[r], value[r]);
    }
    T* to = static_cast<T*>(a.out) + b * a.ob + (int64_t)(h * a.groups + row % a.groups) * a.oh + (int64_t)(row / a.groups) * a.ot + 4 * lane;
    Pack<T, 4> out;
#pragma unroll
    for (int r = 0; r < 4; ++r) out.v[r] = store_cast<T>(total == 0.0f ? 0.0f : finite(value[r] / total));
    if (a.vec_out) {
        store_pack<T, 4>(to, out);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) to[r] = out.v[r];
    }
}

// -------------------------------------------------------------------------------------------------------------- host --
inline bool check_cache(const ahq_kv_cache* cache) {
    if (!cache || !cache->k_codes || !cache->v_codes || !cache->k_amax || !cache->v_amax) return set_error("null cache"), false;
    if (cache->batch <= 0 || cache->heads <= 0 || cache->capacity <= 0) return set_error("bad cache shape"), false;
    if (cache->capacity % kKvTile) return set_error("the capacity must be a multiple of 64 tokens"), false;
    if (cache->capacity > (1 << 30)) return set_error("capacity above 2^30 tokens"), false;
    if ((int64_t)cache->batch * cache->heads > 65535) return set_error("more than 65535 (sequence, head) pairs"), false;
    if (((uintptr_t)cache->k_codes | (uintptr_t)cache->v_codes) % 16) return set_error("cache must be 16-byte aligned"), false;
    return true;
}
inline bool supported(const ahq_kv_cache* cache) {
    if (cache->head_dim != 64 && cache->head_dim != 128 && cache->head_dim != 256)
        return set_error("head sizes are 64, 128 and 256"), false;
    if (cache->block != 16 && cache->block != 32 && cache->block != 64) return set_error("blocks are 16, 32 or 64 tokens"), false;
    return true;
}

template <typename T, int D, int BT>
int launch_append(const KvAppendArgs& a, int64_t bh, int32_t blocks, hipStream_t s) {
    kv_append_kernel<T, D, BT><<<dim3(blocks, (unsigned)bh, 2), kAppendThreads<D, BT>, 0, s>>>(a);
    return check_launch("ahq_kv_append");
}
template <typename T, int D>
int launch_append(const KvAppendArgs& a, int64_t bh, int32_t blocks, int32_t block, hipStream_t s) {
    return block == 16 ? launch_append<T, D, 16>(a, bh, blocks, s)
         : block == 32 ? launch_append<T, D, 32>(a, bh, blocks, s)
                       : launch_append<T, D, 64>(a, bh, blocks, s);
}
template <typename T>
int launch_append(const KvAppendArgs& a, int64_t bh, int32_t blocks, int32_t block, int32_t dim, hipStream_t s) {
    return dim == 64 ? launch_append<T, 64>(a, bh, blocks, block, s)
         : dim == 128 ? launch_append<T, 128>(a, bh, blocks, block, s)
                      : launch_append<T, 256>(a, bh, blocks, block, s);
}

template <typename T, int D>
int launch_values(const KvValuesArgs& a, int64_t bh, hipStream_t s) {
    kv_values_kernel<T, D><<<dim3((a.length + kKvTile - 1) / kKvTile, (unsigned)bh, 2), kBlock, 0, s>>>(a);
    return check_launch("ahq_kv_dequantize");
}
template <typename T>
int launch_values(const KvValuesArgs& a, int64_t bh, int32_t dim, hipStream_t s) {
    return dim == 64 ? launch_values<T, 64>(a, bh, s) : dim == 128 ? launch_values<T, 128>(a, bh, s) : launch_values<T, 256>(a, bh, s);
}

// How a call is shared out.
//
// waves = 0 (kv_attend_kernel): 16 rows to a workgroup, whose four waves share the tokens.  For up to 32 rows, and for more
// where they make little work: fewer than 128 workgroups of the other kind, of at most 2048 token tiles together.
// Otherwise (kv_prompt_kernel) each of four or eight waves has its own 32 rows (float32 queries, 256 channels: 16), so that
// a tile of codes is turned into float16 once for all of them.  Eight share it better; four make more workgroups, which is
// better where they fill the chip once without a split of the token axis, or where a split would cost more than it gives
// (it writes and joins float32 sums, about the time of eight tiles).
//   sequences x heads x groups, queries of tokens, head size   waves 0   4 in one split   8
//   1 x 8 x 4,  64 of 4096, 128                                   24 us            123   35
//   1 x 4 x 4, 512 of 1024, 128                                   19                37   32
//   1 x 8 x 4, 256 of 16384, 128                                 151               467  111
//   1 x 8 x 4, 512 of 512, 128                                    20                22   30
//   1 x 8 x 4, 1024 of 1024, 128                                  41                39   44
//   1 x 8 x 4, 1024 of 4096, 128                                 135               125  107
//   1 x 8 x 4, 2048 of 2048, 128                                 103                73   95
//   2 x 8 x 4, 2048 of 3048, 128                                 321               196  194
//   1 x 8 x 4,  64 of 4096, 128, float32                          22                87   27
//   1 x 8 x 4, 1024 of 4096, 128, float32                        151               132  124
//   1 x 8 x 4,  64 of 4096, 64                                    15                88   26
//   1 x 8 x 4, 512 of 512, 64                                     13                16   21
//   2 x 8 x 4, 512 of 512, 64                                     22                17   24
//   1 x 8 x 4,  64 of 4096, 256                                   46               129   34
//   1 x 8 x 4, 512 of 512, 256                                    58                24   32
//   1 x 8 x 4, 1024 of 4096, 256                                 351               231  169
// The rule is made for 128 channels.  At 256 a workgroup of kv_prompt_kernel takes 128 KB of LDS, so that one runs on a compute
// unit and not two, and the rule is not the best: the first and the last of these rows take 46 and 231 us.
//
// The token axis is split until every compute unit has eight waves, which is what runs there at once with up to 128
// channels, in one round of equal shares with one length for all sequences; where lengths differ (and are known to the
// device alone) shares a third as long even them out.  A share is at least four tiles.
struct AttendPlan { int32_t waves, row_tile, splits, split_tiles; };
inline AttendPlan plan_attend(const ahq_kv_cache* cache, const ahq_kv_queries* q) {
    const int64_t bh = (int64_t)cache->batch * cache->heads, rows = (int64_t)q->queries * (q->query_heads / cache->heads);
    const int64_t tokens = q->lengths ? cache->capacity : q->length_all;
    const int64_t tiles = (tokens + kKvTile - 1) / kKvTile;
    const int wave_rows = q->dtype == AHQ_F32 || cache->head_dim == 256 ? 16 : 32;
    const int64_t of_four = bh * ((rows + 4 * wave_rows - 1) / (4 * wave_rows));
    const bool whole = of_four <= 512 && tiles * (512 - of_four) <= 8 * 512;
    AttendPlan p;
    p.waves = rows <= 32 || (of_four < 128 && of_four * tiles <= 2048) ? 0 : whole ? 4 : 8;
    p.row_tile = p.waves == 0 ? 16 : p.waves * wave_rows;
    const int64_t room = (p.waves == 8 ? 256 : 512) * (q->lengths ? 3 : 1), wgs = bh * ((rows + p.row_tile - 1) / p.row_tile);
    int64_t n = p.waves == 4 ? tiles : (wgs * tiles + room - 1) / room;
    n = (n + 3) / 4 * 4;
    p.split_tiles = (int32_t)(n < 4 ? 4 : n);
    n = (tiles + p.split_tiles - 1) / p.split_tiles;
    p.splits = (int32_t)(n < 1 ? 1 : n);
    return p;
}

template <typename Kernel>
int launch_with_lds(Kernel kernel, const dim3& grid, int threads, size_t lds, const KvAttendArgs& a, hipStream_t s) {
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return set_error(hipGetErrorString(e)), AHQ_ERR_LAUNCH;
    }
    kernel<<<grid, threads, lds, s>>>(a);
    return check_launch("ahq_kv_attend");
}

template <typename T, int D>
int launch_attend(const KvAttendArgs& a, const AttendPlan& p, int64_t bh, hipStream_t s) {
    const dim3 grid((unsigned)bh, (unsigned)((a.rows + p.row_tile - 1) / p.row_tile), (unsigned)p.splits);
    constexpr int NR = sizeof(T) == 4 || D == 256 ? 1 : 2;
    constexpr size_t joined = (size_t)kAttendWaves * (D * 17 + 32) * sizeof(float), buffers = 8 * (size_t)D * kKvTile;
    int rc;
    if (p.waves == 0 && bh * a.capacity * D >= kStreamLoadBytes)
        rc = launch_with_lds(kv_attend_kernel<T, D, true>, grid, kAttendWaves * kWave, joined, a, s);
    else if (p.waves == 0)
        rc = launch_with_lds(kv_attend_kernel<T, D, false>, grid, kAttendWaves * kWave, joined, a, s);
    else if (p.waves == 4)
        rc = launch_with_lds(kv_prompt_kernel<T, D, NR, 4>, grid, 4 * kWave, buffers, a, s);
    else
        rc = launch_with_lds(kv_prompt_kernel<T, D, NR, 8>, grid, 8 * kWave, buffers, a, s);
    if (rc != AHQ_OK || p.splits == 1) return rc;
    if (p.splits <= 8) {
        constexpr int kRows = kJoinThreads / (D / 4);
        kv_join_rows_kernel<T, D><<<dim3((unsigned)((a.rows + kRows - 1) / kRows), (unsigned)bh), kJoinThreads, 0, s>>>(a);
    } else {
        kv_join_kernel<T, D><<<dim3((unsigned)a.rows, (unsigned)bh), kJoinThreads, 0, s>>>(a);
    }
    return check_launch("ahq_kv_attend");
}
template <typename T>
int launch_attend(const KvAttendArgs& a, const AttendPlan& p, int64_t bh, int32_t dim, hipStream_t s) {
    return dim == 64 ? launch_attend<T, 64>(a, p, bh, s) : dim == 128 ? launch_attend<T, 128>(a, p, bh, s) : launch_attend<T, 256>(a, p, bh, s);
}

inline bool attend_shape(const ahq_kv_cache* cache, const ahq_kv_queries* q) {
    if (!q || q->query_heads <= 0 || q->queries < 0) return set_error("bad query shape"), false;
    if (q->query_heads % cache->heads) return set_error("query heads must be a multiple of the cache's heads"), false;
    if ((int64_t)q->queries * (q->query_heads / cache->heads) >= 1ll << 20) return set_error("too many queries in one call"), false;
    return true;
}

}  // namespace ahq

extern "C" int ahq_kv_append(const ahq_kv_cache* cache, const ahq_kv_tokens* x, void* stream) {
    using namespace ahq;
    if (!check_cache(cache)) return AHQ_ERR_INVALID;
    if (!x || x->dtype < AHQ_F32 || x->dtype > AHQ_BF16 || x->tokens < 0) return set_error("bad tokens"), AHQ_ERR_INVALID;
    if (!supported(cache)) return AHQ_ERR_UNSUPPORTED;
    if (x->tokens == 0) return AHQ_OK;
    if (!x->k || !x->v) return set_error("null argument"), AHQ_ERR_INVALID;
    if (x->tokens > (1 << 28)) return set_error("too many tokens"), AHQ_ERR_UNSUPPORTED;
    const int64_t e = x->dtype == AHQ_F32 ? 4 : 2;
    KvAppendArgs a;
    a.x[0] = x->k, a.x[1] = x->v;
    a.vec = 1;
    for (int i = 0; i < 2; ++i) {
        a.sb[i] = x->stride_batch[i], a.sh[i] = x->stride_head[i], a.st[i] = x->stride_token[i];
        if ((uintptr_t)a.x[i] % e) return set_error("misaligned tensor"), AHQ_ERR_INVALID;
        if ((uintptr_t)a.x[i] % 16 || a.sb[i] * e % 16 || a.sh[i] * e % 16 || a.st[i] * e % 16) a.vec = 0;
    }
    a.codes[0] = cache->k_codes, a.codes[1] = cache->v_codes, a.amax[0] = cache->k_amax, a.amax[1] = cache->v_amax;
    a.start = x->start, a.start0 = x->start_all, a.counts = x->counts, a.count0 = x->count_all;
    a.heads = cache->heads, a.tokens = x->tokens, a.capacity = cache->capacity;
    const int64_t bh = (int64_t)cache->batch * cache->heads;
    const int32_t blocks = (x->tokens + cache->block - 2) / cache->block + 1;  // that x->tokens tokens can touch
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (x->dtype == AHQ_F32) return launch_append<float>(a, bh, blocks, cache->block, cache->head_dim, s);
    if (x->dtype == AHQ_F16) return launch_append<f16_t>(a, bh, blocks, cache->block, cache->head_dim, s);
    return launch_append<bf16_t>(a, bh, blocks, cache->block, cache->head_dim, s);
}

extern "C" int ahq_kv_dequantize(const ahq_kv_cache* cache, int32_t dtype, int32_t length, void* k, void* v, void* stream) {
    using namespace ahq;
    if (!check_cache(cache)) return AHQ_ERR_INVALID;
    if (dtype < AHQ_F32 || dtype > AHQ_BF16) return set_error("bad dtype"), AHQ_ERR_INVALID;
    if (length < 0 || length > cache->capacity) return set_error("length outside the cache"), AHQ_ERR_INVALID;
    if (!supported(cache)) return AHQ_ERR_UNSUPPORTED;
    if (length == 0) return AHQ_OK;
    if (length > (1 << 29)) return set_error("more than 2^29 tokens in one call"), AHQ_ERR_UNSUPPORTED;
    if (!k || !v) return set_error("null argument"), AHQ_ERR_INVALID;
    if (((uintptr_t)k | (uintptr_t)v) % 16) return set_error("outputs must be 16-byte aligned"), AHQ_ERR_INVALID;
    KvValuesArgs a;
    a.codes[0] = cache->k_codes, a.codes[1] = cache->v_codes, a.amax[0] = cache->k_amax, a.amax[1] = cache->v_amax;
    a.out[0] = k, a.out[1] = v, a.capacity = cache->capacity, a.length = length, a.block_shift = cache->block == 16 ? 4 : cache->block == 32 ? 5 : 6;
    const int64_t bh = (int64_t)cache->batch * cache->heads;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == AHQ_F32) return launch_values<float>(a, bh, cache->head_dim, s);
    if (dtype == AHQ_F16) return launch_values<f16_t>(a, bh, cache->head_dim, s);
    return launch_values<bf16_t>(a, bh, cache->head_dim, s);
}

extern "C" size_t ahq_kv_attend_workspace_bytes(const ahq_kv_cache* cache, const ahq_kv_queries* q) {
    using namespace ahq;
    if (!check_cache(cache) || !attend_shape(cache, q) || !supported(cache) || q->queries == 0) return 0;
    const AttendPlan p = plan_attend(cache, q);
    if (p.splits == 1) return 0;
    const size_t rows = (size_t)cache->batch * cache->heads * q->queries * (q->query_heads / cache->heads);
    return rows * p.splits * (cache->head_dim + 2) * sizeof(float);
}

extern "C" int ahq_kv_attend(const ahq_kv_cache* cache, const ahq_kv_queries* q, void* workspace, size_t workspace_bytes,
                             void* stream) {
    using namespace ahq;
    if (!check_cache(cache) || !attend_shape(cache, q)) return AHQ_ERR_INVALID;
    if (q->dtype < AHQ_F32 || q->dtype > AHQ_BF16) return set_error("bad dtype"), AHQ_ERR_INVALID;
    if (!supported(cache)) return AHQ_ERR_UNSUPPORTED;
    if (q->queries == 0) return AHQ_OK;
    if (!q->q || !q->out) return set_error("null argument"), AHQ_ERR_INVALID;
    if (!(q->scale > -0x1p126f && q->scale < 0x1p126f)) return set_error("the scale must be finite"), AHQ_ERR_INVALID;
    const size_t need = ahq_kv_attend_workspace_bytes(cache, q);
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return set_error("workspace too small"), AHQ_ERR_WORKSPACE;
    const int64_t e = q->dtype == AHQ_F32 ? 4 : 2;
    if (((uintptr_t)q->q | (uintptr_t)q->out) % e) return set_error("misaligned tensor"), AHQ_ERR_INVALID;
    const int64_t bh = (int64_t)cache->batch * cache->heads;
    const AttendPlan p = plan_attend(cache, q);
    if (p.splits > 65535) return set_error("too many splits of the token axis"), AHQ_ERR_UNSUPPORTED;
    KvAttendArgs a;
    a.q = q->q, a.out = q->out;
    a.qb = q->q_stride_batch, a.qh = q->q_stride_head, a.qt = q->q_stride_query;
    a.ob = q->out_stride_batch, a.oh = q->out_stride_head, a.ot = q->out_stride_query;
    a.k_codes = cache->k_codes, a.v_codes = cache->v_codes, a.k_amax = cache->k_amax, a.v_amax = cache->v_amax;
    a.lengths = q->lengths, a.counts = q->counts, a.length0 = q->length_all, a.count0 = q->count_all;
    a.heads = cache->heads, a.groups = q->query_heads / cache->heads, a.queries = q->queries;
    a.capacity = cache->capacity, a.block_shift = cache->block == 16 ? 4 : cache->block == 32 ? 5 : 6;
    a.rows = a.queries * a.groups, a.row_tile = p.row_tile, a.splits = p.splits, a.split_tiles = p.split_tiles;
    a.scale = q->scale * 1.44269504088896340736f;
    a.vec = (uintptr_t)q->q % 16 == 0 && a.qb * e % 16 == 0 && a.qh * e % 16 == 0 && a.qt * e % 16 == 0;
    a.vec_out = (uintptr_t)q->out % (4 * e) == 0 && a.ob % 4 == 0 && a.oh % 4 == 0 && a.ot % 4 == 0;
    a.part = static_cast<float*>(workspace);
    a.part_stat = a.part + (size_t)bh * a.rows * a.splits * cache->head_dim;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (q->dtype == AHQ_F32) return launch_attend<float>(a, p, bh, cache->head_dim, s);
    if (q->dtype == AHQ_F16) return launch_attend<f16_t>(a, p, bh, cache->head_dim, s);
    return launch_attend<bf16_t>(a, p, bh, cache->head_dim, s);
}
