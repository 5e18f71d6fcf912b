// Linear layers on packed 4-bit weights.
//
//   y[m, n] = sum_g s[n, g] * ( sum_{k in g} x[m, k] * (u[n, k] + z[n, g]) ) + b[n]
//
// u are the codes counted from the lower end of their grid (0..15), z = offset + qmin + zero-point shift, s the float32
// scale of the group.  The inner sums run on the matrix cores with both factors exact: u is a whole number that
// bfloat16 and float16 hold, x is used as it is (float32 as a sum of three bfloat16 parts), the accumulators are
// float32.  z is taken out of the inner sum as z * sum(x), where sum(x) is one more matrix instruction against ones, and
// added to the group's sum in float32.  The scale multiplies the finished group sum in float32, so
// the only rounding to fewer bits is the one of y.  An infinite x makes its row NaN (0 * inf and inf - inf both occur).
//
// Weight layout: tiles of 16 rows x 128 columns, 1 KB each, along a row of tiles first.  Lane 16 c + i of the wave that
// owns a tile finds its 16 bytes at 16 * lane: word j holds row i, columns 32 j + 8 c + e, e = 0..3 in the low and 4..7
// in the high halves of bytes 0..3.  A code in the low half of a zero byte is the float8 (e4m3) number u * 2^-9, normal
// or not, so v_cvt_scalef32_pk_*_fp8 with the scale 512 turns two codes into two exact 16-bit floats: 7 vector
// instructions for 8 codes.

#include "../../include/aimet_amd_serving.h"
#include "ahq_host.h"
#include "mma.h"

namespace ahq {

constexpr int kTileRows = 16;
constexpr int kTileCols = 128;
constexpr int kTileBytes = 1024;

// -------------------------------------------------------------------------------------------------------- fragments --
template <typename T> struct Int4Traits;
typedef float f32x8 __attribute__((ext_vector_type(8), aligned(16)));
template <> struct Int4Traits<bf16_t> { typedef bf16x8 Frag; typedef u32x4_t Raw; static constexpr int kParts = 1; };
template <> struct Int4Traits<f16_t> { typedef f16x8 Frag; typedef u32x4_t Raw; static constexpr int kParts = 1; };
template <> struct Int4Traits<float> { typedef bf16x8 Frag; typedef f32x8 Raw; static constexpr int kParts = 3; };

template <typename Frag> __device__ __forceinline__ Frag decode_codes(uint32_t w);
template <> __device__ __forceinline__ bf16x8 decode_codes<bf16x8>(uint32_t w) {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    union { bf16x2 h[4]; bf16x8 v; } r;
    r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false);
    r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true);
    r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false);
    r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true);
    return r.v;
}
template <> __device__ __forceinline__ f16x8 decode_codes<f16x8>(uint32_t w) {
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    union { f16x2 h[4]; f16x8 v; } r;
    r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, false);
    r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 512.0f, true);
    r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, false);
    r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 512.0f, true);
    return r.v;
}

template <typename Frag> __device__ __forceinline__ Frag ones_fragment();
template <> __device__ __forceinline__ bf16x8 ones_fragment<bf16x8>() {
    const uint32_t w = 0x3f803f80u;
    return __builtin_bit_cast(bf16x8, u32x4_t{w, w, w, w});
}
template <> __device__ __forceinline__ f16x8 ones_fragment<f16x8>() {
    const uint32_t w = 0x3c003c00u;
    return __builtin_bit_cast(f16x8, u32x4_t{w, w, w, w});
}

// Eight activations from column k on; columns from `cols` on count as zero.  `vec`: rows start on 16-byte boundaries.
template <typename T>
__device__ __forceinline__ typename Int4Traits<T>::Raw load_raw(const T* __restrict__ row, int64_t k, int64_t cols, bool vec) {
    typename Int4Traits<T>::Raw w = {};
    if constexpr (sizeof(T) == 2) {
        if (vec && k + 8 <= cols) {
            w = *reinterpret_cast<const u32x4_t*>(row + k);
        } else if (k < cols) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + e < cols) w[e / 2] |= (uint32_t)row[k + e].bits << (16 * (e & 1));
        }
    } else {
        if (vec && k + 8 <= cols) {
            w = *reinterpret_cast<const f32x8*>(row + k);
        } else if (k < cols) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (k + e < cols) w[e] = row[k + e];
        }
    }
    return w;
}
template <typename T>
__device__ __forceinline__ void raw_to_fragments(const typename Int4Traits<T>::Raw& w, typename Int4Traits<T>::Frag* out) {
    if constexpr (sizeof(T) == 2) {
        out[0] = __builtin_bit_cast(typename Int4Traits<T>::Frag, w);
    } else {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = w[e];
        split_bf16<3>(v, out);
    }
}

struct Int4Args {
    const void* x;
    const uint8_t* w;
    const float* scale;   // [row tile][groups][16]
    const int8_t* zero;   // same layout, or null: z = zero_const everywhere
    const void* bias;
    void* y;
    int64_t m, n, k, ldx, ldy;
    int64_t tiles;          // 128-column tiles of a row
    int64_t ntiles;         // tiles of 16 rows
    int64_t groups;
    uint64_t fold_inverse;  // ceil(2^32 / folds per group)
    float zero_const;
    int32_t vec_x;
};

// ------------------------------------------------------------------------------------------------------- few activations --
// Decoding: one to a few tokens.  One workgroup of 16 waves to a compute unit; `splits` waves share a row tile and take its
// 128-column tiles in turn, so a workgroup owns 16 / splits row tiles.  Activations wait in LDS (CHUNKED: `turns` turns of
// the waves at a time) and are the A operand here, the weight's rows the columns of the result: a lane's results belong to
// one channel, whose scale and zero point are one register.  Bound by the stream of codes, so a wave asks for kDepth tiles
// at once, right behind its share of the activations; those are read back from LDS, whose waits do not hold up the stream.
//
// The activations' sums are formed along with the products, by every wave for itself: matrix instructions wait for nobody
// here, and a pass of their own with its barrier took 0.4 to 0.8 us (32 x 4096 x 4096 14.0 -> 12.4 us).
//
// One token x 14336 x 4096 (33 MB): 10.9 us, 3.0 TB/s, of which the start takes 4.1 (launch 2.0, activations).  One, three and
// four tiles at once instead of two: 12.0, 11.3, 11.7 us; two workgroups on a compute unit (64 registers): 17 us, spills.
constexpr int kLdsWaves = 16;
constexpr int kLdsThreads = kLdsWaves * kWave;
constexpr int kFewRows = 32;

template <typename T, int FOLD, int MT, bool ASYM, bool CHUNKED>
__global__ __launch_bounds__(kLdsThreads) void int4_linear_lds_kernel(Int4Args a, int splits, int turns, int row_bytes) {
    typedef typename Int4Traits<T>::Frag Frag;
    constexpr int P = Int4Traits<T>::kParts;
    constexpr int kFolds = 4 / FOLD, kDepth = 2;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int i = lane & 15, c = lane >> 4;
    // 32 activations to a workgroup; more are further workgroups' (blockIdx.y)
    const int64_t m0 = (int64_t)blockIdx.y * kFewRows;
    const int m = a.m - m0 < kFewRows ? (int)(a.m - m0) : kFewRows;
    const int tiles = (int)a.tiles, groups = (int)a.groups;
    const int per_group = kLdsWaves / splits;
    const int split = wave % splits;
    const int64_t tile = (int64_t)blockIdx.x * per_group + wave / splits;
    extern __shared__ u32x4_t lds[];
    char* xs = reinterpret_cast<char*>(lds);

    // activations of `held` tiles from tile `from` on: [part][row][columns], rows padded by 16 bytes so that 16 of them lie
    // on different banks
    const int held = CHUNKED ? turns * splits : tiles;
    const int chunks = held * 16, total = m * chunks;
    int from = 0;
    const auto fetch = [&](int id) {
        const int row = id / chunks;
        return load_raw<T>(static_cast<const T*>(a.x) + (m0 + row) * a.ldx, (CHUNKED ? from * kTileCols : 0) + (id - row * chunks) * 8, a.k, a.vec_x);
    };
    const auto put = [&](int id, const typename Int4Traits<T>::Raw& raw) {
        const int row = id / chunks;
        Frag f[P];
        raw_to_fragments<T>(raw, f);
#pragma unroll
        for (int p = 0; p < P; ++p)
            *reinterpret_cast<Frag*>(xs + (p * m + row) * row_bytes + (id - row * chunks) * 16) = f[p];
    };
    // all but the last kBatch rounds are stored at once; those wait until the first codes have been asked for
    constexpr int kBatch = sizeof(T) == 2 ? 4 : 2;
    typename Int4Traits<T>::Raw raw[kBatch];
    int id;
    const auto begin_activations = [&] {
        for (id = threadIdx.x; id + kBatch * kLdsThreads < total; id += kBatch * kLdsThreads) {
#pragma unroll
            for (int u = 0; u < kBatch; ++u) raw[u] = fetch(id + u * kLdsThreads);
#pragma unroll
            for (int u = 0; u < kBatch; ++u) put(id + u * kLdsThreads, raw[u]);
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (id + u * kLdsThreads < total) raw[u] = fetch(id + u * kLdsThreads);
    };
    const auto end_activations = [&] {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (id + u * kLdsThreads < total) put(id + u * kLdsThreads, raw[u]);
        __syncthreads();
    };
    begin_activations();

    const bool live = tile < a.ntiles;
    const int64_t tile_at = live ? tile : a.ntiles - 1;
    const u32x4_t* wp = reinterpret_cast<const u32x4_t*>(a.w + tile_at * a.tiles * kTileBytes) + lane;
    const float* sp = a.scale + tile_at * a.groups * kTileRows + i;
    const int8_t* zp = ASYM ? a.zero + tile_at * a.groups * kTileRows + i : nullptr;
    u32x4_t w[kDepth];
    float scale[kDepth][kFolds];
    int zero[kDepth][kFolds];
    const auto load = [&](int d, int kt) {
        w[d] = __builtin_nontemporal_load(wp + kt * (kTileBytes / 16));
#pragma unroll
        for (int f = 0; f < kFolds; ++f) {
            int g = (int)(((uint64_t)(unsigned)(kt * kFolds + f) * a.fold_inverse) >> 32);
            g = g < groups ? g : groups - 1;
            scale[d][f] = sp[g * kTileRows];
            if constexpr (ASYM) zero[d][f] = zp[g * kTileRows];
        }
    };
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
        if (split + d * splits < tiles) load(d, split + d * splits);
    end_activations();

    f32x4 acc[MT];
    const char* xrow[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        acc[mt] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int row = 16 * mt + i;  // rows behind the last one repeat it and are not stored
        xrow[mt] = xs + (row < m ? row : m - 1) * row_bytes + 16 * c;
    }
    const Frag ones = ones_fragment<Frag>();
    // CHUNKED: as many turns for every wave, since they meet at barriers
    const int end = CHUNKED ? (tiles + splits - 1) / splits * splits : tiles;
    int left = turns;  // that the activations in LDS serve
    for (int kt0 = split; kt0 < end; kt0 += kDepth * splits) {
#pragma unroll
        for (int d = 0; d < kDepth; ++d) {
            const int kt = kt0 + d * splits;
            if constexpr (CHUNKED) {
                if (left == 0 && kt < end) {
                    __syncthreads();
                    from = kt - split, left = turns;
                    begin_activations();
                    end_activations();
                }
                --left;
            }
            if (kt < tiles) {
                const int at = CHUNKED ? kt - from : kt;
#pragma unroll
                for (int f = 0; f < kFolds; ++f) {
                    Frag wf[FOLD];
#pragma unroll
                    for (int j = 0; j < FOLD; ++j) wf[j] = decode_codes<Frag>(w[d][f * FOLD + j]);
                    const float z = ASYM ? a.zero_const + (float)zero[d][f] : a.zero_const;
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) {
                        f32x4 sum = {0.f, 0.f, 0.f, 0.f}, part = sum;  // of the activations, and of the products
#pragma unroll
                        for (int j = 0; j < FOLD; ++j)
#pragma unroll
                            for (int p = 0; p < P; ++p) {
                                const Frag x = *reinterpret_cast<const Frag*>(xrow[mt] + p * m * row_bytes + at * 256 + (f * FOLD + j) * 64);
                                part = mma(x, wf[j], part);
                                sum = mma(x, ones, sum);
                            }
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            acc[mt][r] = __builtin_fmaf(scale[d][f], __builtin_fmaf(z, sum[r], part[r]), acc[mt][r]);
                    }
                }
                if (kt + kDepth * splits < tiles) load(d, kt + kDepth * splits);
            }
        }
    }

    f32x4* red = reinterpret_cast<f32x4*>(lds);  // [wave][MT][64], over the activations
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) red[(wave * MT + mt) * kWave + lane] = acc[mt];
    __syncthreads();
    for (int o = threadIdx.x; o < per_group * MT * kWave; o += kLdsThreads) {
        const int unit = o / (MT * kWave), q = o % (MT * kWave);
        const int64_t n = ((int64_t)blockIdx.x * per_group + unit) * kTileRows + (q & 15);
        const int row = q / kWave * 16 + (q >> 4 & 3) * 4;
        if (n >= a.n || row >= m) continue;
        f32x4 v = red[unit * splits * MT * kWave + q];
        for (int s = 1; s < splits; ++s) {
            const f32x4 u = red[(unit * splits + s) * MT * kWave + q];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += u[r];
        }
        const float b = a.bias ? load_f32(static_cast<const T*>(a.bias)[n]) : 0.0f;
        T* y = static_cast<T*>(a.y) + (m0 + row) * a.ldy + n;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (row + r < m) y[r * a.ldy] = store_cast<T>(v[r] + b);
    }
}

// ------------------------------------------------------------------------------------------------------ many activations --
// Prompts.  A workgroup computes 16 * MT activations x 64 * NW channels with eight waves: NW side by side times 8 / NW groups
// that take steps of 128 or 64 columns of the row in turn, each with activations of its own in LDS (two buffers, in the order of
// the matrix operands), so that two waves on each SIMD overlap matrix and vector work and a 2048 x 2048 result already
// fills the chip.  Per step and wave: 8 * MT matrix instructions, 56 vector instructions to turn codes into
// operands and 16 * MT to scale the finished group sums (every 64 columns at least): the two kinds nearly balance.  The
// wave that brings activations in sums them, with one matrix instruction a fragment.  The groups' results are added
// through LDS, in a fixed order.
//
// Bound by the issue of vector instructions next to the matrix ones.  2048 x 2048 x 8192 bfloat16: 83 us, 830 TFLOP/s;
// 300 x 4096 x 4096 float16 with zero points: 33.5 us.  Codes asked for four steps ahead instead of two: 107 us (spills).
constexpr int kManyWaves = 8;

// NW waves side by side (of 64 channels each), 8 / NW groups along the row.
template <typename T, int MT, int NW> struct ManyLayout {
    static constexpr int kParts = Int4Traits<T>::kParts;
    static constexpr int kGroups = kManyWaves / NW;
    static constexpr int kDeep = kParts == 1 && NW == 4 ? 4 : 2;      // matrix instructions along a step: 128 or 64 columns
    static constexpr int kStage = kDeep * MT * kParts * kWave;        // operands (16 bytes) of a step
    static constexpr int kSums = kDeep * MT * 4;                      // f32x4 of its folds' sums
    static constexpr size_t kBytes = (size_t)kGroups * 2 * (kStage + kSums) * 16;
    static constexpr size_t kJoin = (size_t)(kGroups / 2) * NW * MT * 4 * kWave * 16;
    static constexpr size_t kLds = kBytes > kJoin ? kBytes : kJoin;
};

// The values of the wave's four rows of 16 lanes, each for all of them.
__device__ __forceinline__ void rows_of(uint32_t v, float* out) {
    const auto pair = __builtin_amdgcn_permlane16_swap(v, v, false, false);  // rows 0 0 2 2 and 1 1 3 3
    const auto even = __builtin_amdgcn_permlane32_swap(pair[0], pair[0], false, false);
    const auto odd = __builtin_amdgcn_permlane32_swap(pair[1], pair[1], false, false);
    out[0] = bits_to_f32(even[0]), out[1] = bits_to_f32(odd[0]), out[2] = bits_to_f32(even[1]), out[3] = bits_to_f32(odd[1]);
}

// WHOLE: rows start on 16-byte boundaries and are whole steps long, so that no load has to be looked at.
template <typename T, int FOLD, int MT, int NW, bool ASYM, bool WHOLE>
__global__ __launch_bounds__(kManyWaves * kWave, 2) void int4_linear_many_kernel(Int4Args a, int mblocks, int nblocks) {
    typedef typename Int4Traits<T>::Frag Frag;
    typedef ManyLayout<T, MT, NW> Layout;
    constexpr int kGroups = Layout::kGroups;
    constexpr int P = Int4Traits<T>::kParts;
    constexpr int NT = 4;                  // row tiles of a wave
    constexpr int kDeep = Layout::kDeep, kCols = 32 * kDeep;
    constexpr int kFolds = kDeep / FOLD;   // of a step
    typedef uint32_t Words __attribute__((ext_vector_type(kDeep)));
    constexpr int kMine = MT / NW;         // activation tiles that a wave brings in
    static_assert(MT % NW == 0, "each wave brings in as many");
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int i = lane & 15, c = lane >> 4;
    const int side = wave % NW, group = wave / NW;
    // Blocks on one XCD (every eighth workgroup) form a band of four activation blocks: they share activations and
    // weights in its L2.
    const int total = mblocks * nblocks, per_xcd = (total + 7) / 8;
    const int order = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
    if (order >= total || (int)(blockIdx.x >> 3) >= per_xcd) return;
    const int band = order / (4 * nblocks), band_rows = mblocks - 4 * band < 4 ? mblocks - 4 * band : 4;
    const int in_band = order - band * 4 * nblocks;
    const int mblock = 4 * band + in_band % band_rows, nblock = in_band / band_rows;
    const int64_t m0 = (int64_t)mblock * (16 * MT);
    const int64_t tile0 = (int64_t)nblock * (NW * NT) + side * NT;

    extern __shared__ u32x4_t lds[];
    Frag* stages = reinterpret_cast<Frag*>(lds) + (size_t)group * 2 * Layout::kStage;
    f32x4* sums = reinterpret_cast<f32x4*>(lds) + (size_t)kGroups * 2 * Layout::kStage + group * 2 * Layout::kSums;

    // Rows behind the last one repeat it and are not stored.  WHOLE: a scalar base and 32-bit offsets of the lane.
    const T* rows[kMine];
    uint32_t row_at[kMine];
    const char* block = static_cast<const char*>(a.x) + m0 * a.ldx * (int64_t)sizeof(T);
#pragma unroll
    for (int t = 0; t < kMine; ++t) {
        const int r = 16 * (side * kMine + t) + i, in = m0 + r < a.m ? r : (int)(a.m - 1 - m0);
        if constexpr (WHOLE) row_at[t] = (uint32_t)((in * (int)a.ldx + 8 * c) * (int)sizeof(T));
        else rows[t] = static_cast<const T*>(a.x) + (m0 + in) * a.ldx;
    }
    // scalar bases; the lane's offset is added at the load
    const uint8_t* wp[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) wp[nt] = a.w + (tile0 + nt < a.ntiles ? tile0 + nt : a.ntiles - 1) * a.tiles * kTileBytes;
    // lane 16 c + i brings in the scale of channel i of row tile c; rows_of() hands it to all lanes of column i
    const int64_t scale_at = (tile0 + c < a.ntiles ? tile0 + c : a.ntiles - 1) * a.groups * kTileRows + i;
    const float* sp = a.scale + scale_at;
    const int8_t* zp = ASYM ? a.zero + scale_at : nullptr;
    const int steps = (int)((a.k + kCols - 1) / kCols), groups = (int)a.groups;
    const int rounds = (steps + kGroups - 1) / kGroups;  // the same for all waves: they meet at barriers

    typename Int4Traits<T>::Raw raw[kMine][kDeep];
    const auto fetch = [&](int step) {
#pragma unroll
        for (int t = 0; t < kMine; ++t)
#pragma unroll
            for (int j = 0; j < kDeep; ++j) {
                if constexpr (WHOLE)
                    raw[t][j] = *reinterpret_cast<const typename Int4Traits<T>::Raw*>(block + (int64_t)step * (kCols * sizeof(T)) + row_at[t] + 32 * j * sizeof(T));
                else
                    raw[t][j] = load_raw<T>(rows[t], (int64_t)step * kCols + 32 * j + 8 * c, a.k, a.vec_x);
            }
    };
    const Frag ones = ones_fragment<Frag>();
    const auto put = [&](int buffer) {
#pragma unroll
        for (int t = 0; t < kMine; ++t) {
            const int mt = side * kMine + t;
#pragma unroll
            for (int f = 0; f < kFolds; ++f) {
                f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = f * FOLD; j < (f + 1) * FOLD; ++j) {
                    Frag x[P];
                    raw_to_fragments<T>(raw[t][j], x);
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        stages[buffer * Layout::kStage + ((j * MT + mt) * P + p) * kWave + lane] = x[p];
                        part = mma(x[p], ones, part);
                    }
                }
                if constexpr (!ASYM) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) part[r] *= a.zero_const;
                }
                if (i == 0) sums[buffer * Layout::kSums + (f * MT + mt) * 4 + c] = part;
            }
        }
    };
    f32x4 acc[MT][NT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Codes, scales and activations are asked for two steps before their use.
    Words next_w[2][NT];
    uint32_t next_scale[2][kFolds];
    int next_zero[2][kFolds];
    const auto fetch_weight = [&](int q, int step) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
            next_w[q][nt] = *reinterpret_cast<const Words*>(wp[nt] + (int64_t)(step * kDeep / 4) * kTileBytes + step * kDeep % 4 * 4 + (uint32_t)(lane * 16));
#pragma unroll
        for (int f = 0; f < kFolds; ++f) {
            int g = (int)(((uint64_t)(unsigned)(step * kFolds + f) * a.fold_inverse) >> 32);
            g = g < groups ? g : groups - 1;
            next_scale[q][f] = f32_to_bits(sp[(int64_t)g * kTileRows]);
            if constexpr (ASYM) next_zero[q][f] = zp[(int64_t)g * kTileRows];
        }
    };
    // The workgroups of a band start at four places of the row, so that they do not ask the same memory channels at once.
    const int turn = (mblock & 3) * rounds / 4;
    const auto step_of = [&](int n) {  // this group's n-th step; may lie behind the row's end
        const int r = n + turn;
        return (r < rounds ? r : r - rounds) * kGroups + group;
    };
    const auto at_most = [&](int step) { return step < steps ? step : steps - 1; };
    fetch(at_most(step_of(0)));
    fetch_weight(0, at_most(step_of(0)));
    put(0);
    fetch(at_most(step_of(rounds > 1 ? 1 : 0)));
    fetch_weight(1, at_most(step_of(rounds > 1 ? 1 : 0)));
    const auto work = [&](int n, int s) {  // the two buffers take turns: s = n % 2
        // one barrier a step: what is read behind it was stored in front of it; what is stored behind it goes where the
        // last reads were in front of it
        __syncthreads();
        const bool live = step_of(n) < steps;  // behind the row's end there is nothing to add
        Words w[NT];
        float scale[kFolds][NT], zero[kFolds][NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) w[nt] = next_w[s][nt];
#pragma unroll
        for (int f = 0; f < kFolds; ++f) {
            rows_of(live ? next_scale[s][f] : 0u, scale[f]);
            if constexpr (ASYM) rows_of(f32_to_bits(a.zero_const + (float)next_zero[s][f]), zero[f]);
        }
        fetch_weight(s, at_most(step_of(n + 2 < rounds ? n + 2 : n)));
        // operands of the next activation tile are read while this one's products run, in an order that is kept
        Frag xf[2][FOLD][P], wf[NT][FOLD];
        f32x4 sum[2];
        const auto read = [&](int at) {
            const int f = at / MT, mt = at % MT;
#pragma unroll
            for (int j = 0; j < FOLD; ++j)
#pragma unroll
                for (int p = 0; p < P; ++p)
                    xf[at & 1][j][p] = stages[s * Layout::kStage + (((f * FOLD + j) * MT + mt) * P + p) * kWave + lane];
            sum[at & 1] = sums[s * Layout::kSums + (f * MT + mt) * 4 + c];
        };
        read(0);
#pragma unroll
        for (int at = 0; at < kFolds * MT; ++at) {
            const int f = at / MT, mt = at % MT;
            if (mt == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < FOLD; ++j) wf[nt][j] = decode_codes<Frag>(w[nt][f * FOLD + j]);
            }
            if (at == kFolds * MT / 2) {  // half way: the next step's activations have come
                put(s ^ 1);
                fetch(at_most(step_of(n + 2 < rounds ? n + 2 : n)));
            }
            if (at + 1 < kFolds * MT) read(at + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                f32x4 part = sum[at & 1];
                if constexpr (ASYM) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) part[r] *= zero[f][nt];
                }
#pragma unroll
                for (int j = 0; j < FOLD; ++j)
#pragma unroll
                    for (int p = 0; p < P; ++p) part = mma(xf[at & 1][j][p], wf[nt][j], part);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[mt][nt][r] = __builtin_fmaf(scale[f][nt], part[r], acc[mt][nt][r]);
                asm volatile("" : "+v"(acc[mt][nt]));  // the sum is formed here, not with all others at the end
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int n = 0; n < rounds; n += 2) {
        work(n, 0);
        if (n + 1 < rounds) work(n + 1, 1);
    }

    // the upper half of the groups hands its sums to the lower one, until one group has them all
    f32x4* join = reinterpret_cast<f32x4*>(lds);
#pragma unroll
    for (int far = kGroups / 2; far >= 1; far /= 2) {
        __syncthreads();
        if (group >= far && group < 2 * far) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) join[(((group - far) * NW + side) * MT * NT + mt * NT + nt) * kWave + lane] = acc[mt][nt];
        }
        __syncthreads();
        if (group < far) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const f32x4 u = join[((group * NW + side) * MT * NT + mt * NT + nt) * kWave + lane];
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[mt][nt][r] += u[r];
                }
        }
    }
    if (group) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int64_t n = (tile0 + nt) * kTileRows + i;
        if (n >= a.n) continue;
        const float b = a.bias ? load_f32(static_cast<const T*>(a.bias)[n]) : 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t m = m0 + 16 * mt + 4 * c + r;
                if (m < a.m) static_cast<T*>(a.y)[m * a.ldy + n] = store_cast<T>(acc[mt][nt][r] + b);
            }
    }
}

// ----------------------------------------------------------------------------------------------------------- packing --
__global__ __launch_bounds__(kBlock) void int4_pack_kernel(const int8_t* __restrict__ codes, int64_t n, int64_t k,
                                                           int32_t qmin, int64_t tiles, int64_t words,
                                                           uint32_t* __restrict__ out) {
    const int64_t id = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (id >= words) return;
    const int j = (int)(id & 3), lane = (int)((id >> 2) & 63);
    const int64_t tile = id >> 8;
    const int64_t row = tile / tiles * kTileRows + (lane & 15);
    const int64_t col = tile % tiles * kTileCols + 32 * j + 8 * (lane >> 4);
    uint32_t w = 0;
    if (row < n) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (col + e >= k) break;
            const uint32_t u = (uint32_t)(codes[row * k + col + e] - qmin) & 15u;
            w |= u << (e < 4 ? 8 * e : 8 * (e - 4) + 4);
        }
    }
    out[id] = w;
}

// ------------------------------------------------------------------------------------------------------------- host --
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How the kernel of few activations shares a call out: waves to a row tile, turns whose activations LDS holds at a time,
// bytes of LDS.
struct LdsPlan { int splits, turns, row_bytes; bool chunked; size_t lds; int64_t blocks, slices; };
inline LdsPlan plan_lds(const Int4Args& a, int parts, int mt) {
    LdsPlan p;
    const int64_t m = a.m < kFewRows ? a.m : kFewRows;
    p.slices = ceil_div(a.m, kFewRows);
    // as many waves to a row tile as one workgroup on each of the 256 compute units gives
    p.splits = kLdsWaves;
    while (p.splits > 1 && (p.splits > a.tiles || ceil_div(a.ntiles, kLdsWaves / p.splits) > 256)) p.splits /= 2;
    const int64_t fit = (160 * 1024 - m * parts * 16) / (m * parts * 256);  // 13 tiles at least: 16 activations in three parts
    while (p.splits > 1 && p.splits > fit) p.splits /= 2;
    const int64_t all = ceil_div(a.tiles, p.splits), most = fit / p.splits;
    p.chunked = a.tiles > fit;
    p.turns = (int)ceil_div(all, ceil_div(all, most));  // even shares
    const int64_t held = p.chunked ? p.turns * p.splits : a.tiles;
    p.row_bytes = (int)(held * 256 + 16);
    const size_t red = (size_t)kLdsWaves * 1024 * mt, bytes = (size_t)(m * parts * p.row_bytes);
    p.lds = bytes > red ? bytes : red;
    p.blocks = ceil_div(a.ntiles, kLdsWaves / p.splits);
    return p;
}

template <typename T, int FOLD, int MT, bool ASYM, bool CHUNKED>
int launch_lds(const Int4Args& a, const LdsPlan& p, hipStream_t stream) {
    const auto kernel = int4_linear_lds_kernel<T, FOLD, MT, ASYM, CHUNKED>;
    if (p.lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds);
        if (e != hipSuccess) return set_error(hipGetErrorString(e)), AHQ_ERR_LAUNCH;
    }
    kernel<<<dim3((unsigned)p.blocks, (unsigned)p.slices), kLdsThreads, p.lds, stream>>>(a, p.splits, p.turns, p.row_bytes);
    return check_launch("ahq_int4_linear");
}
template <typename T, int FOLD, int MT>
int launch_lds(const Int4Args& a, const LdsPlan& p, hipStream_t stream) {
    if (p.chunked) return a.zero ? launch_lds<T, FOLD, MT, true, true>(a, p, stream) : launch_lds<T, FOLD, MT, false, true>(a, p, stream);
    return a.zero ? launch_lds<T, FOLD, MT, true, false>(a, p, stream) : launch_lds<T, FOLD, MT, false, false>(a, p, stream);
}

template <typename T, int FOLD, int MT, int NW, bool ASYM, bool WHOLE>
int launch_many(const Int4Args& a, hipStream_t stream) {
    constexpr size_t lds = ManyLayout<T, MT, NW>::kLds;
    const auto kernel = int4_linear_many_kernel<T, FOLD, MT, NW, ASYM, WHOLE>;
    if (lds > 65536) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return set_error(hipGetErrorString(e)), AHQ_ERR_LAUNCH;
    }
    const int64_t mblocks = ceil_div(a.m, 16 * MT), nblocks = ceil_div(a.n, 64 * NW);
    if (mblocks * nblocks > (1 << 22)) return set_error("too many activations and channels in one call"), AHQ_ERR_UNSUPPORTED;
    kernel<<<(unsigned)(ceil_div(mblocks * nblocks, 8) * 8), kManyWaves * kWave, lds, stream>>>(a, (int)mblocks, (int)nblocks);
    return check_launch("ahq_int4_linear");
}
template <typename T, int FOLD, int MT, int NW>
int launch_many(const Int4Args& a, hipStream_t stream) {
    const bool whole = a.vec_x && a.k % (32 * ManyLayout<T, MT, NW>::kDeep) == 0 && a.ldx * (int64_t)sizeof(T) * 16 * MT < (1ll << 31);
    if (a.zero) return whole ? launch_many<T, FOLD, MT, NW, true, true>(a, stream) : launch_many<T, FOLD, MT, NW, true, false>(a, stream);
    return whole ? launch_many<T, FOLD, MT, NW, false, true>(a, stream) : launch_many<T, FOLD, MT, NW, false, false>(a, stream);
}

template <typename T, int FOLD>
int launch_linear(Int4Args a, int64_t group, hipStream_t stream) {
    // folds per group
    const auto folds = [&](int64_t columns) {
        const uint64_t n = group == a.k ? 1ull << 32 : (uint64_t)(group / columns);
        a.fold_inverse = ((1ull << 32) + n - 1) / n;
    };
    // Few activations: against the smallest blocks below, 32 x 4096 x 4096 12.4 and 16.5 us, 32 x 4096 x 14336 35 and 38 us.
    // More, 32 to a workgroup, while all of these run at once: 64 x 2048 x 2048 8.1 us against 11.2, 128 x 1000 x 8192 22 and 25,
    // 300 x 400 x 14336 37 and 38.  float32, whose three parts take as much more room, up to 16: 16 x 4096 x 4096 15 us against
    // 17, 12 x 4096 x 14336 31 and 44, but 20 x 4096 x 4096 19 and 18, 32 x 4096 x 4096 33 and 18.
    const LdsPlan p = plan_lds(a, Int4Traits<T>::kParts, a.m <= 16 ? 1 : 2);
    if (a.m <= 16) {
        folds(32 * FOLD);
        return launch_lds<T, FOLD, 1>(a, p, stream);
    }
    if constexpr (sizeof(T) == 2) {
        if (a.m <= kFewRows || p.blocks * p.slices <= 256) {
            folds(32 * FOLD);
            return launch_lds<T, FOLD, 2>(a, p, stream);
        }
    }
    constexpr int kFold = FOLD == 1 ? 1 : 2;
    folds(32 * kFold);
    const auto one_round = [&](int64_t rows, int64_t channels) { return ceil_div(a.m, rows) * ceil_div(a.n, channels) <= 256; };
    if constexpr (sizeof(T) == 2) {
        // The smallest block whose workgroups still run on the 256 compute units all at once, else the largest: a block's time
        // hardly depends on how many others run, and it grows more slowly than its size.  At 4096 x 4096, in the order 32 x 64,
        // 32 x 128, 64 x 128, 64 x 256: 64 activations 17, 21, 29, 40 us; 256: 31, 23, 30, 41; 512: -, 40, 31, 41;
        // 640: -, 56, 57, 41.
        if (one_round(32, 64)) return launch_many<T, kFold, 2, 1>(a, stream);
        if (one_round(32, 128)) return launch_many<T, kFold, 2, 2>(a, stream);
        if (one_round(64, 128)) return launch_many<T, kFold, 4, 2>(a, stream);
        return launch_many<T, kFold, 4, 4>(a, stream);
    } else {
        // in the order 16 x 64, 32 x 128 (three parts fill LDS): 64 x 1000 x 8192 28 and 60 us, 64 x 4096 x 4096 34 in the second
        if (one_round(16, 64)) return launch_many<T, kFold, 1, 1>(a, stream);
        return launch_many<T, kFold, 2, 2>(a, stream);
    }
}

template <typename T>
int launch_linear(const Int4Args& a, int64_t group, hipStream_t stream) {
    // The scale is applied every 32, 64 or 128 columns: as rarely as one scale lasts (128 keeps the group sums short
    // where a scale covers a whole row).
    if (group == a.k || group % 128 == 0) return launch_linear<T, 4>(a, group, stream);
    if (group % 64 == 0) return launch_linear<T, 2>(a, group, stream);
    return launch_linear<T, 1>(a, group, stream);
}

}  // namespace ahq

extern "C" size_t ahq_int4_packed_bytes(int64_t n, int64_t k) {
    if (n <= 0 || k <= 0 || n > (1ll << 28) || k > (1ll << 20)) return 0;
    return (size_t)(ahq::ceil_div(n, ahq::kTileRows) * ahq::ceil_div(k, ahq::kTileCols) * ahq::kTileBytes);
}

extern "C" int ahq_int4_pack(const int8_t* codes, int64_t n, int64_t k, int32_t qmin, void* packed, void* stream) {
    using namespace ahq;
    if (!codes || !packed) return set_error("null argument"), AHQ_ERR_INVALID;
    if (ahq_int4_packed_bytes(n, k) == 0) return set_error("bad weight shape"), AHQ_ERR_INVALID;
    if (qmin < -128 || qmin > 112) return set_error("qmin outside [-128, 112]"), AHQ_ERR_INVALID;
    if ((uintptr_t)packed % 16) return set_error("packed weights must be 16-byte aligned"), AHQ_ERR_INVALID;
    const int64_t tiles = ceil_div(k, kTileCols), words = (int64_t)ahq_int4_packed_bytes(n, k) / 4;
    if (words > 0xffffff00ll) return set_error("weight too large"), AHQ_ERR_UNSUPPORTED;
    int4_pack_kernel<<<(unsigned)ceil_div(words, kBlock), kBlock, 0, static_cast<hipStream_t>(stream)>>>(
        codes, n, k, qmin, tiles, words, static_cast<uint32_t*>(packed));
    return check_launch("ahq_int4_pack");
}

extern "C" int ahq_int4_linear(const ahq_int4_weight* w, int32_t dtype, const void* x, int64_t m, int64_t ldx,
                               const void* bias, void* y, int64_t ldy, void* stream) {
    using namespace ahq;
    if (!w || !w->packed || !w->scale) return set_error("null weight"), AHQ_ERR_INVALID;
    const int64_t n = w->n, k = w->k, group = w->group;
    if (dtype < AHQ_F32 || dtype > AHQ_BF16) return set_error("bad dtype"), AHQ_ERR_INVALID;
    if (m < 0 || ahq_int4_packed_bytes(n, k) == 0) return set_error("bad shape"), AHQ_ERR_INVALID;
    if (group <= 0 || group > k || k % group) return set_error("the group must divide the row"), AHQ_ERR_INVALID;
    if (group != k && group % 32) return set_error("groups are multiples of 32 columns or the whole row"), AHQ_ERR_UNSUPPORTED;
    if (((uintptr_t)w->packed | (uintptr_t)w->scale | (uintptr_t)w->zero) % 16)
        return set_error("packed weights, scales and zero points must be 16-byte aligned"), AHQ_ERR_INVALID;
    if (m == 0) return AHQ_OK;
    if (!x || !y) return set_error("null argument"), AHQ_ERR_INVALID;
    if (ldx < k || ldy < n) return set_error("row strides smaller than the rows"), AHQ_ERR_INVALID;
    const size_t e = dtype == AHQ_F32 ? 4 : 2;
    if (((uintptr_t)x | (uintptr_t)y | (uintptr_t)bias) % e) return set_error("misaligned tensor"), AHQ_ERR_INVALID;
    if (m > (1ll << 20)) return set_error("more than 2^20 activations in one call"), AHQ_ERR_UNSUPPORTED;
    Int4Args a;
    a.x = x, a.w = static_cast<const uint8_t*>(w->packed), a.scale = w->scale, a.zero = w->zero, a.bias = bias, a.y = y;
    a.m = m, a.n = n, a.k = k, a.ldx = ldx, a.ldy = ldy;
    a.tiles = ceil_div(k, kTileCols), a.ntiles = ceil_div(n, kTileRows), a.groups = k / group;
    a.zero_const = w->zero_const;
    a.vec_x = (uintptr_t)x % 16 == 0 && (ldx * (int64_t)e) % 16 == 0;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == AHQ_F32) return launch_linear<float>(a, group, s);
    if (dtype == AHQ_F16) return launch_linear<f16_t>(a, group, s);
    return launch_linear<bf16_t>(a, group, s);
}
