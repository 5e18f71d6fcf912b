// A key/value cache held in 8 bits, and the attention that reads it.
//
// Stored: codes in [-127, 127] and, for every block of `block` tokens (16, 32 or 64) of a sequence and head, the largest
// magnitude `amax` among them; a code stands for code * amax / 127.  Keys lie as [sequence, head, token, channel].  Values
// lie as [sequence, head, tile of 64 tokens, channel, token of the tile]: the product of the probabilities and the values
// sums over tokens, and a lane of a matrix instruction then finds the 16 tokens it needs of one channel in one 16-byte
// load.
//
// Writing (kv_append_kernel): a workgroup owns one block of one head.  amax = max(what the block had, |new tokens|), code =
// rint(127 x / amax), half to even and exact; where amax grows, the codes the block had become rint(code * old / new).
//
// Reading (kv_attend_kernel): one pass over the tokens with the running maximum and sum of the softmax.  Rows of a tile
// are the query heads of one key head (and the queries behind each other, where there are several).  A wave takes 64
// tokens at a time: scores = keys (A) x queries (B) on the matrix cores, so that lane 16 c + i of the result holds 16
// tokens of row i.  Keys are handed to the instruction in an order that makes those the tokens 16 c .. 16 c + 15 of the
// tile: that is the B operand of the next product, values (A) x probabilities (B), without any exchange between lanes.
// Codes are exact in bfloat16; queries are used exactly (float16 as two, float32 as three bfloat16 parts); the block's
// scales multiply scores and probabilities in float32; the probabilities enter the second product as two bfloat16 parts
// (16 bits, 2^-17 relative) for 16-bit queries and as three for float32 ones.  Everything else is float32.

#include "../../include/aimet_amd_serving.h"
#include "ahq_host.h"
#include "mma.h"

namespace ahq {

constexpr int kKvTile = 64;

// ------------------------------------------------------------------------------------------------------------ append --
struct KvAppendArgs {
    const void* x[2];        // new keys, new values
    int64_t sb[2], sh[2], st[2];  // strides in elements: sequence, head, token
    int8_t* codes[2];
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

// rint(127 v / amax), half to even, exact.  Fast form: with amax and 127 v exact in few bits, the remainder of the
// approximate quotient is exact in float32 and says which neighbour is nearer; otherwise float64, whose quotient of
// these operands (31 and 24 bits) is correctly rounded and therefore falls on the right side of every border.
struct CodeRule {
    float amax, inverse;
    bool fast;
};
__device__ __forceinline__ CodeRule code_rule(float amax, bool narrow) {
    CodeRule r;
    r.amax = amax;
    r.fast = narrow && amax > 1e-30f && amax < 1e36f && (f32_to_bits(amax) & 0x1fffu) == 0;
    r.inverse = r.fast ? 127.0f / amax : 0.0f;
    return r;
}
__device__ __forceinline__ int to_code(float v, const CodeRule& rule) {
    if (!(rule.amax > 0.0f) || v != v) return 0;
    float q;
    if (rule.fast) {
        v = fminf(fmaxf(v, -rule.amax), rule.amax);
        q = __builtin_rintf(v * rule.inverse);
        const float twice = 2.0f * __builtin_fmaf(-q, rule.amax, 127.0f * v);
        const bool odd = ((int)q & 1) != 0;
        if (twice > rule.amax || (odd && twice == rule.amax)) q += 1.0f;
        if (twice < -rule.amax || (odd && twice == -rule.amax)) q -= 1.0f;
    } else {
        const double w = fmin(fmax((double)v, -(double)rule.amax), (double)rule.amax);
        q = (float)__builtin_rint(127.0 * w / (double)rule.amax);
    }
    return (int)q;
}

// VEC elements per thread and step, one step per thread; THREADS = block * D / 8 capped at 512, ITEMS steps.
template <typename T, int D, int BT>
__global__ __launch_bounds__(BT * D / 8 < 512 ? BT * D / 8 : 512) void kv_append_kernel(KvAppendArgs a) {
    constexpr int kVecs = BT * D / 8;
    constexpr int kThreads = kVecs < 512 ? kVecs : 512;
    constexpr int kItems = kVecs / kThreads;
    constexpr int kPitch = BT + 4;
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

    const T* x = static_cast<const T*>(a.x[which]) + b * a.sb[which] + h * a.sh[which];
    float v[kItems][8];
    float top = 0.0f;
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const int id = it * kThreads + threadIdx.x, t = id / (D / 8), d = id % (D / 8) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[it][e] = 0.0f;
        if (t >= old_end && t < new_end) {
            const T* row = x + (int64_t)(p0 + t - range.begin) * a.st[which] + d;
            if (a.vec) {
                constexpr int kPer = 16 / sizeof(T);
#pragma unroll
                for (int u = 0; u < 8 / kPer; ++u) {
                    const Pack<T, kPer> w = load_pack<T, kPer>(row + u * kPer);
#pragma unroll
                    for (int e = 0; e < kPer; ++e) v[it][u * kPer + e] = load_f32(w.v[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[it][e] = load_f32(row[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, finite_magnitude(v[it][e]));
    }
    __shared__ float part[kThreads / kWave];
    top = wave_reduce(top, OpMaxF());
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = top;
    float* amax_at = a.amax[which] + (int64_t)bh * (a.capacity / BT) + blk;
    const float before = old_end > 0 ? *amax_at : 0.0f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) top = fmaxf(top, part[w]);
    const float amax = fmaxf(before, top);
    const bool rescale = old_end > 0 && amax > before;
    const CodeRule rule = code_rule(amax, sizeof(T) == 2);
    const int first = rescale ? 0 : old_end;  // first token whose codes are stored

    int8_t* keys = a.codes[which] + ((int64_t)bh * a.capacity + p0) * D;
    // tile of 64 tokens that holds this block, and the block's place in it
    int8_t* tile = a.codes[which] + ((int64_t)bh * a.capacity + p0 / kKvTile * kKvTile) * D + p0 % kKvTile;
    __shared__ alignas(16) int8_t stage[D * kPitch];
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const int id = it * kThreads + threadIdx.x, t = id / (D / 8), d = id % (D / 8) * 8;
        if (t < first || t >= new_end) continue;
        union { int8_t b[8]; u32x2_t w; } out;
        if (t >= old_end) {
#pragma unroll
            for (int e = 0; e < 8; ++e) out.b[e] = (int8_t)to_code(v[it][e], rule);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int q = which ? tile[(d + e) * kKvTile + t] : keys[(int64_t)t * D + d + e];
                out.b[e] = (int8_t)(int)__builtin_rint((double)q * (double)before / (double)amax);
            }
        }
        if (which == 0) {
            *reinterpret_cast<u32x2_t*>(keys + (int64_t)t * D + d) = out.w;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) stage[(d + e) * kPitch + t] = out.b[e];
        }
    }
    if (which == 1) {
        __syncthreads();
        for (int id = threadIdx.x; id < D * (BT / 16); id += kThreads) {
            const int d = id / (BT / 16), t = id % (BT / 16) * 16;
            const uint32_t* from = reinterpret_cast<const uint32_t*>(stage + d * kPitch + t);
            int8_t* to = tile + d * kKvTile + t;
            if (first <= t && t + 16 <= new_end) {
                *reinterpret_cast<u32x4_t*>(to) = u32x4_t{from[0], from[1], from[2], from[3]};
            } else {
                for (int e = 0; e < 16; ++e)
                    if (t + e >= first && t + e < new_end) to[e] = stage[d * kPitch + t + e];
            }
        }
    }
    // read by other threads before the first barrier above, so it is written behind the last one
    if (threadIdx.x == 0) *amax_at = amax;
}

// -------------------------------------------------------------------------------------------------------- dequantize --
struct KvValuesArgs {
    const int8_t* codes[2];
    const float* amax[2];
    void* out[2];  // [sequence, head, length, D]
    int32_t capacity, length, block;
};

template <typename T, int D>
__global__ __launch_bounds__(kBlock) void kv_values_kernel(KvValuesArgs a) {
    constexpr int kPitch = kKvTile + 4;
    const int which = blockIdx.z, tile = blockIdx.x;
    const int64_t bh = blockIdx.y;
    const int p0 = tile * kKvTile;
    const int8_t* codes = a.codes[which] + (bh * a.capacity + p0) * D;
    const float* amax = a.amax[which] + bh * (a.capacity / a.block);
    T* out = static_cast<T*>(a.out[which]) + (bh * a.length + p0) * D;
    __shared__ alignas(16) int8_t stage[D * kPitch];
    if (which) {
        for (int id = threadIdx.x; id < D * 4; id += kBlock) {
            const u32x4_t w = *reinterpret_cast<const u32x4_t*>(codes + id * 16);
            uint32_t* to = reinterpret_cast<uint32_t*>(stage + id / 4 * kPitch + id % 4 * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e) to[e] = w[e];
        }
        __syncthreads();
    }
    for (int id = threadIdx.x; id < kKvTile * (D / 8); id += kBlock) {
        const int t = id / (D / 8), d = id % (D / 8) * 8;
        if (p0 + t >= a.length) break;
        const float s = amax[(p0 + t) / a.block] / 127.0f;
        union { int8_t b[8]; u32x2_t w; } in;
        if (which) {
#pragma unroll
            for (int e = 0; e < 8; ++e) in.b[e] = stage[(d + e) * kPitch + t];
        } else {
            in.w = *reinterpret_cast<const u32x2_t*>(codes + (int64_t)t * D + d);
        }
        constexpr int kPer = 16 / sizeof(T);
#pragma unroll
        for (int u = 0; u < 8 / kPer; ++u) {
            Pack<T, kPer> w;
#pragma unroll
            for (int e = 0; e < kPer; ++e) w.v[e] = store_cast<T>((float)in.b[u * kPer + e] * s);
            store_pack<T, kPer>(out + (int64_t)t * D + d + u * kPer, w);
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ attend --
struct KvAttendArgs {
    const void* q;
    void* out;
    int64_t qb, qh, qt, ob, oh, ot;  // strides in elements
    const int8_t *k_codes, *v_codes;
    const float *k_amax, *v_amax;
    const int32_t* lengths;  // null: length0
    const int32_t* counts;   // null: count0
    int32_t length0, count0;
    int32_t heads, groups, queries, capacity, block;
    int32_t row_tiles, splits;
    float scale;             // of the scores, times log2(e)
    int32_t vec;             // rows of q start on 16-byte boundaries
    float* part;             // [sequence * head][row tile][split][16][D], then [..][16][2]: maximum and sum
    float* part_stat;
};

template <typename T> struct AttendTraits;
template <> struct AttendTraits<bf16_t> { static constexpr int kQ = 1, kP = 2; };
template <> struct AttendTraits<f16_t> { static constexpr int kQ = 2, kP = 2; };
template <> struct AttendTraits<float> { static constexpr int kQ = 3, kP = 3; };

// Eight codes as bfloat16: whole numbers up to 127 have no low half in float32.
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t a, uint32_t b) {
    u32x4_t w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        w[e] = pack_high_halves((float)(int8_t)(a >> (16 * e)), (float)(int8_t)(a >> (16 * e + 8)));
        w[2 + e] = pack_high_halves((float)(int8_t)(b >> (16 * e)), (float)(int8_t)(b >> (16 * e + 8)));
    }
    return __builtin_bit_cast(bf16x8, w);
}

template <typename T, int N>
__device__ __forceinline__ void load_query(const T* p, bool live, bool vec, bf16x8* out) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (live) {
        constexpr int kPer = 16 / sizeof(T);
        if (vec) {
#pragma unroll
            for (int u = 0; u < 8 / kPer; ++u) {
                const Pack<T, kPer> w = load_pack<T, kPer>(p + u * kPer);
#pragma unroll
                for (int e = 0; e < kPer; ++e) v[u * kPer + e] = load_f32(w.v[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = load_f32(p[e]);
        }
    }
    split_bf16<N>(v, out);
}

struct SequenceView { int length, count; };
__device__ __forceinline__ SequenceView view_sequence(const KvAttendArgs& a, int b) {
    int n = a.lengths ? a.lengths[b] : a.length0;
    int t = a.counts ? a.counts[b] : a.count0;
    n = n < 0 ? 0 : n > a.capacity ? a.capacity : n;
    t = t < 0 ? 0 : t > a.queries ? a.queries : t;
    return {n, t};
}

constexpr int kAttendWaves = 4;

template <typename T, int D>
__global__ __launch_bounds__(kAttendWaves * kWave) void kv_attend_kernel(KvAttendArgs a) {
    constexpr int NQ = AttendTraits<T>::kQ, NP = AttendTraits<T>::kP;
    constexpr int kSteps = D / 32;   // matrix instructions along the channels
    constexpr int kOut = D / 16;     // output tiles of 16 channels
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int i = lane & 15, c = lane >> 4;
    const int split = blockIdx.x, row_tile = blockIdx.y;
    const int64_t bh = blockIdx.z;
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
    const SequenceView seq = view_sequence(a, b);

    const int rows = a.queries * a.groups;
    const int row = row_tile * 16 + i;
    const int t = row / a.groups;
    // the last token this row sees; below 0: none
    const int last = row < rows && t < seq.count ? seq.length - seq.count + t : -1;
    int t_end = (row_tile * 16 + 15) / a.groups;
    if (t_end >= seq.count) t_end = seq.count - 1;
    const int seen = seq.length - seq.count + t_end + 1;  // tokens the tile's last row sees
    const int tiles = t_end < 0 || seen <= 0 ? 0 : (seen + kKvTile - 1) / kKvTile;
    const int per_split = (tiles + a.splits - 1) / a.splits;
    const int first = split * per_split;
    const int stop = first + per_split < tiles ? first + per_split : tiles;

    bf16x8 q[kSteps][NQ];
    {
        const bool live = last >= 0;
        const T* base = static_cast<const T*>(a.q) + b * a.qb + (int64_t)(h * a.groups + row % a.groups) * a.qh + (int64_t)t * a.qt;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) load_query<T, NQ>(base + 64 * (s / 2) + 16 * c + 8 * (s % 2), live, a.vec, q[s]);
    }
    f32x4 o[kOut];
#pragma unroll
    for (int u = 0; u < kOut; ++u) o[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    float top = -__builtin_inff(), sum = 0.0f;

    const int8_t* keys = a.k_codes + bh * a.capacity * D;
    const int8_t* values = a.v_codes + bh * a.capacity * D;
    const float* k_amax = a.k_amax + bh * (a.capacity / a.block);
    const float* v_amax = a.v_amax + bh * (a.capacity / a.block);
    const int key_row = (i >> 2) * 16 + (i & 3);  // token of A row i in the score tile s: key_row + 4 s

    for (int tile = first + wave; tile < stop; tile += kAttendWaves) {
        const int p0 = tile * kKvTile;
        u32x4_t kw[4][D / 64];
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int u = 0; u < D / 64; ++u)
                kw[s][u] = *reinterpret_cast<const u32x4_t*>(keys + (int64_t)(p0 + key_row + 4 * s) * D + 64 * u + 16 * c);
        const int block_at = (p0 + 16 * c) / a.block;
        const float k_scale = k_amax[block_at] / 127.0f * a.scale;
        const float v_scale = v_amax[block_at] / 127.0f;
        float sc[16];
        float tile_top = -__builtin_inff();
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < kSteps; ++u) {
                const u32x4_t w = kw[s][u / 2];
                const bf16x8 kf = u % 2 ? codes_to_bf16(w[2], w[3]) : codes_to_bf16(w[0], w[1]);
#pragma unroll
                for (int p = 0; p < NQ; ++p) acc = mma(kf, q[u][p], acc);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float v = p0 + 16 * c + 4 * s + r <= last ? acc[r] * k_scale : -__builtin_inff();
                sc[4 * s + r] = v;
                tile_top = fmaxf(tile_top, v);
            }
        }
        tile_top = fmaxf(tile_top, __shfl_xor(tile_top, 16, kWave));
        tile_top = fmaxf(tile_top, __shfl_xor(tile_top, 32, kWave));
        const float now = fmaxf(top, tile_top);
        const float base = now == -__builtin_inff() ? 0.0f : now;
        const float fade = __builtin_amdgcn_exp2f(top - base);
        top = now;
        sum *= fade;
#pragma unroll
        for (int u = 0; u < kOut; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[u][r] *= fade;
        bf16x8 pf[2][NP];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool hidden = p0 + 16 * c + 8 * w + e > last;
                const float v = hidden ? 0.0f : __builtin_amdgcn_exp2f(sc[8 * w + e] - base);
                sum += v;
                p[e] = hidden ? 0.0f : v * v_scale;
            }
            split_bf16<NP>(p, pf[w]);
        }
#pragma unroll
        for (int u = 0; u < kOut; ++u) {
            const u32x4_t w = *reinterpret_cast<const u32x4_t*>(values + (int64_t)p0 * D + (16 * u + i) * kKvTile + 16 * c);
            const bf16x8 v0 = codes_to_bf16(w[0], w[1]), v1 = codes_to_bf16(w[2], w[3]);
#pragma unroll
            for (int p = 0; p < NP; ++p) o[u] = mma(v0, pf[0][p], o[u]);
#pragma unroll
            for (int p = 0; p < NP; ++p) o[u] = mma(v1, pf[1][p], o[u]);
        }
    }
    sum += __shfl_xor(sum, 16, kWave);
    sum += __shfl_xor(sum, 32, kWave);

    // the waves' results are joined through LDS, in wave order
    constexpr int kPitch = 17;
    extern __shared__ float joined[];  // [wave][D][17], then [wave][16][2]
    float* stats = joined + kAttendWaves * D * kPitch;
#pragma unroll
    for (int u = 0; u < kOut; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) joined[(wave * D + 16 * u + 4 * c + r) * kPitch + i] = o[u][r];
    if (c == 0) stats[(wave * 16 + i) * 2] = top, stats[(wave * 16 + i) * 2 + 1] = sum;
    __syncthreads();
    for (int id = threadIdx.x; id < 16 * D; id += kAttendWaves * kWave) {
        const int rr = id / D, d = id % D;
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
        const int out_row = row_tile * 16 + rr;
        if (out_row >= rows) continue;
        if (a.splits == 1) {
            T* to = static_cast<T*>(a.out) + b * a.ob + (int64_t)(h * a.groups + out_row % a.groups) * a.oh + (int64_t)(out_row / a.groups) * a.ot;
            to[d] = store_cast<T>(total == 0.0f ? 0.0f : value / total);
        } else {
            const int64_t at = ((bh * a.row_tiles + row_tile) * a.splits + split) * 16 + rr;
            a.part[at * D + d] = value;
            if (d == 0) a.part_stat[at * 2] = best, a.part_stat[at * 2 + 1] = total;
        }
    }
}

// One workgroup per row: the splits' results are added in their order.
template <typename T, int D>
__global__ __launch_bounds__(D) void kv_join_kernel(KvAttendArgs a) {
    const int row = blockIdx.x, d = threadIdx.x;
    const int64_t bh = blockIdx.y;
    const int b = (int)(bh / a.heads), h = (int)(bh % a.heads);
    const int64_t at = (bh * a.row_tiles + row / 16) * a.splits * 16 + row % 16;
    float best = -__builtin_inff();
    for (int s = 0; s < a.splits; ++s) best = fmaxf(best, a.part_stat[(at + (int64_t)s * 16) * 2]);
    const float base = best == -__builtin_inff() ? 0.0f : best;
    float total = 0.0f, value = 0.0f;
    for (int s = 0; s < a.splits; ++s) {
        const float f = __builtin_amdgcn_exp2f(a.part_stat[(at + (int64_t)s * 16) * 2] - base);
        total += f * a.part_stat[(at + (int64_t)s * 16) * 2 + 1];
        value += f * a.part[(at + (int64_t)s * 16) * D + d];
    }
    T* to = static_cast<T*>(a.out) + b * a.ob + (int64_t)(h * a.groups + row % a.groups) * a.oh + (int64_t)(row / a.groups) * a.ot;
    to[d] = store_cast<T>(total == 0.0f ? 0.0f : value / total);
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
    constexpr int kVecs = BT * D / 8;
    kv_append_kernel<T, D, BT><<<dim3(blocks, (unsigned)bh, 2), kVecs < 512 ? kVecs : 512, 0, s>>>(a);
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

// Splits of the token axis: enough workgroups to fill the chip four times over, at least four tiles (one for each wave)
// to a split.
inline int32_t attend_splits(int64_t bh, int64_t row_tiles, int64_t tokens) {
    const int64_t tiles = (tokens + kKvTile - 1) / kKvTile;
    int64_t n = (1024 + bh * row_tiles - 1) / (bh * row_tiles);
    const int64_t most = (tiles + kAttendWaves - 1) / kAttendWaves;
    n = n > most ? most : n;
    return (int32_t)(n < 1 ? 1 : n);
}

template <typename T, int D>
int launch_attend(const KvAttendArgs& a, int64_t bh, hipStream_t s) {
    constexpr size_t lds = (size_t)kAttendWaves * (D * 17 + 32) * sizeof(float);
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kv_attend_kernel<T, D>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return set_error(hipGetErrorString(e)), AHQ_ERR_LAUNCH;
    }
    kv_attend_kernel<T, D><<<dim3(a.splits, a.row_tiles, (unsigned)bh), kAttendWaves * kWave, lds, s>>>(a);
    const int rc = check_launch("ahq_kv_attend");
    if (rc != AHQ_OK || a.splits == 1) return rc;
    kv_join_kernel<T, D><<<dim3(a.queries * a.groups, (unsigned)bh), D, 0, s>>>(a);
    return check_launch("ahq_kv_attend");
}
template <typename T>
int launch_attend(const KvAttendArgs& a, int64_t bh, int32_t dim, hipStream_t s) {
    return dim == 64 ? launch_attend<T, 64>(a, bh, s) : dim == 128 ? launch_attend<T, 128>(a, bh, s) : launch_attend<T, 256>(a, bh, s);
}

inline bool attend_shape(const ahq_kv_cache* cache, const ahq_kv_queries* q) {
    if (!q || q->query_heads <= 0 || q->queries < 0) return set_error("bad query shape"), false;
    if (q->query_heads % cache->heads) return set_error("query heads must be a multiple of the cache's heads"), false;
    if ((int64_t)q->queries * (q->query_heads / cache->heads) > 65535ll * 16) return set_error("too many queries in one call"), false;
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
    if (x->tokens > (1 << 29)) return set_error("too many tokens"), AHQ_ERR_UNSUPPORTED;
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
    if (!k || !v) return set_error("null argument"), AHQ_ERR_INVALID;
    if (((uintptr_t)k | (uintptr_t)v) % 16) return set_error("outputs must be 16-byte aligned"), AHQ_ERR_INVALID;
    KvValuesArgs a;
    a.codes[0] = cache->k_codes, a.codes[1] = cache->v_codes, a.amax[0] = cache->k_amax, a.amax[1] = cache->v_amax;
    a.out[0] = k, a.out[1] = v, a.capacity = cache->capacity, a.length = length, a.block = cache->block;
    const int64_t bh = (int64_t)cache->batch * cache->heads;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == AHQ_F32) return launch_values<float>(a, bh, cache->head_dim, s);
    if (dtype == AHQ_F16) return launch_values<f16_t>(a, bh, cache->head_dim, s);
    return launch_values<bf16_t>(a, bh, cache->head_dim, s);
}

extern "C" size_t ahq_kv_attend_workspace_bytes(const ahq_kv_cache* cache, const ahq_kv_queries* q) {
    using namespace ahq;
    if (!check_cache(cache) || !attend_shape(cache, q) || !supported(cache) || q->queries == 0) return 0;
    const int64_t bh = (int64_t)cache->batch * cache->heads;
    const int64_t row_tiles = ((int64_t)q->queries * (q->query_heads / cache->heads) + 15) / 16;
    const int32_t splits = attend_splits(bh, row_tiles, q->lengths ? cache->capacity : q->length_all);
    return splits == 1 ? 0 : (size_t)(bh * row_tiles * splits * 16) * (cache->head_dim + 2) * sizeof(float);
}

extern "C" int ahq_kv_attend(const ahq_kv_cache* cache, const ahq_kv_queries* q, void* workspace, size_t workspace_bytes,
                             void* stream) {
    using namespace ahq;
    if (!check_cache(cache) || !attend_shape(cache, q)) return AHQ_ERR_INVALID;
    if (q->dtype < AHQ_F32 || q->dtype > AHQ_BF16) return set_error("bad dtype"), AHQ_ERR_INVALID;
    if (!supported(cache)) return AHQ_ERR_UNSUPPORTED;
    if (q->queries == 0) return AHQ_OK;
    if (!q->q || !q->out) return set_error("null argument"), AHQ_ERR_INVALID;
    const size_t need = ahq_kv_attend_workspace_bytes(cache, q);
    if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
        return set_error("workspace too small"), AHQ_ERR_WORKSPACE;
    const int64_t e = q->dtype == AHQ_F32 ? 4 : 2;
    if (((uintptr_t)q->q | (uintptr_t)q->out) % e) return set_error("misaligned tensor"), AHQ_ERR_INVALID;
    const int64_t bh = (int64_t)cache->batch * cache->heads;
    KvAttendArgs a;
    a.q = q->q, a.out = q->out;
    a.qb = q->q_stride_batch, a.qh = q->q_stride_head, a.qt = q->q_stride_query;
    a.ob = q->out_stride_batch, a.oh = q->out_stride_head, a.ot = q->out_stride_query;
    a.k_codes = cache->k_codes, a.v_codes = cache->v_codes, a.k_amax = cache->k_amax, a.v_amax = cache->v_amax;
    a.lengths = q->lengths, a.counts = q->counts, a.length0 = q->length_all, a.count0 = q->count_all;
    a.heads = cache->heads, a.groups = q->query_heads / cache->heads, a.queries = q->queries;
    a.capacity = cache->capacity, a.block = cache->block;
    a.row_tiles = (int32_t)(((int64_t)a.queries * a.groups + 15) / 16);
    a.splits = attend_splits(bh, a.row_tiles, q->lengths ? cache->capacity : q->length_all);
    a.scale = q->scale * 1.44269504088896340736f;
    a.vec = (uintptr_t)q->q % 16 == 0 && a.qb * e % 16 == 0 && a.qh * e % 16 == 0 && a.qt * e % 16 == 0;
    a.part = static_cast<float*>(workspace);
    a.part_stat = a.part + (size_t)bh * a.row_tiles * a.splits * 16 * cache->head_dim;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (q->dtype == AHQ_F32) return launch_attend<float>(a, bh, cache->head_dim, s);
    if (q->dtype == AHQ_F16) return launch_attend<f16_t>(a, bh, cache->head_dim, s);
    return launch_attend<bf16_t>(a, bh, cache->head_dim, s);
}
