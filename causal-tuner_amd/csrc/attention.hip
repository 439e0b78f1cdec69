// Attention over packed records on gfx950: forward, and the backward that recomputes the
// probabilities. Per record and head, with query i and key j of the record,
//   s_ij = scale q_i . k_j          visible: j < limit_i = keys (plain) or
//                                   min(keys, i + 1 + keys - queries) (causal)
//   p_ij = exp(s_ij - m_i) / l_i,  m_i = max_j s_ij,  l_i = sum_j exp(s_ij - m_i),  o_i = sum_j p_ij v_j
//   delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i)
//   dv_j = sum_i p_ij do_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j
// (the place of the reference's kernels/attention.py:58-93, which calls a library).
//
// Rows. The `group` query heads of one key/value head are rows of one matrix: row r of a
// record is token r / group, head r % group. One tile of keys then serves all heads of the
// group, a single token of a shared head already fills rows, and the key gradients' sum
// over heads is the sum over rows.
//
// Matrix products. Every product is v_mfma_*_32x32x* with the wave's own rows (forward and
// dq) or keys (dk, dv) as the column index, so lane l holds column l % 32 of the scores and
// 16 of their 32 rows: softmax statistics are one register per lane, the probabilities go
// from the accumulators straight into the next product's B operand (rounded to bf16 in
// pairs; the operands' k order follows the accumulator's), and the outputs o^T, dq^T, dk^T
// and dv^T accumulate 32 rows of the head dimension at a time. The A operands come from
// LDS: rows as stored (ds_read_b128) for the scores, transposed (ds_read_b64_tr_b16) for
// the outputs.
//
// Rounding. Scores, statistics, delta and all sums are fp32. bf16 inputs round p and ds to
// bf16 for the second products, which take bf16 (each value off by at most 2^-8 of itself, as
// the output's own rounding: together 1.4 times the output's, 0.0024 against 0.0017 in norm);
// float32 inputs round nothing. Where a row sees few keys, do . v and delta nearly cancel, and
// a delta from the rounded output made dq and dk 0.005 off (records of one to four tokens): the
// output is divided by the sum of the p that entered its product (the backward has the exact one), and
// for a backward the forward keeps the output's rounding error in bf16 as well (`rest`).
//
// dq and dk/dv are two kernels that each recompute s (7 products instead of 5): the one-pass
// form would add dq over workgroups by atomics, whose order changes results from run to run,
// or through a partial dq per key tile, whose traffic (4.3 GB written and read at 8192 rows of
// 32 heads) outweighs the two products.
//
// What bounds it. The matrix instructions and, beside them, the exponentials: 8192 causal rows
// of 32 heads of 128 over one key/value head, bf16: forward 613 us (897 TFLOP/s; 10 us of it for
// the second sum and `rest`), dq 782 (1055), dk and dv 1351 (814), with the matrix instructions
// busy 42, 52 and 35% of the SIMDs' cycles. Large library products reach 1100 to 1600 on the same
// card by size and layout; HBM traffic is a few percent. Few query tokens: the stream of keys and
// values, 131072 keys of 8 heads in 103 us, 5.2 TB/s (a large copy 5.2).
// Tried and left out: the two waves of a SIMD in turns (one in matrix instructions while the
// other has its exponentials, two barriers a step): forward 615 -> 580 us, but 43 -> 46 at three
// short records and both backward kernels slower; 8 waves per forward workgroup (7% slower at
// short records); scores of the next step before the current step's exponentials in the forward.

#include <math.h>

#include <algorithm>
#include <type_traits>
#include <vector>

#include "gemm_common.hpp"

namespace ct {
namespace {

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

constexpr int kThreads = 256;   // 4 waves
constexpr int kWaveCols = 32;   // rows (forward, dq) or keys (dk, dv) per wave
constexpr int kTile = 128;      // per workgroup
constexpr int kRowWaves = 4, kRowTile = kWaveCols * kRowWaves;   // of a forward or dq workgroup
constexpr int kEntry = 8;       // int32 per plan entry
constexpr float kLog2e = 1.4426950408889634f;

struct Record {
    int64_t q_start, q_len, k_start, k_len;
};

// A plan: pieces of work, joins of what was cut, and the workgroups' lists of pieces.
struct Item {
    int32_t record, begin;  // first row (forward, dq) or key (dk, dv) of the tile
    int32_t lo, hi;         // piece: its keys or rows; join: its first partial and their number
    int32_t slot;           // piece: its partial, or -1 for the whole tile; join: first row in the tile
    int32_t rows;           // join: rows or keys
    int32_t pad0, pad1;
};

struct Group {
    int32_t first, count, pad[6];
};

struct AttnParams {
    const char *q, *k, *v, *out, *dout;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // bytes
    int64_t o_token, o_head;                                    // bytes: out, dq (contiguous)
    int64_t do_token, do_head;                                  // bytes
    const Record *records;
    const Item *items;
    const Group *groups;
    char *dst0, *dst1;    // out | dq | dk, dv
    char *rest;           // out's rounding error, as out, or null
    int64_t d_token;      // bytes between tokens of dst0 and dst1
    float2 *stats;        // [tokens, heads] Running's m and log2 of the sum (+inf where a row sees no key)
    float4 *terms;        // [tokens, heads] what dq leaves of a row for dk and dv: sstat's three, 1 where far
    float *part0, *part1; // split partials
    int32_t heads, kv_heads, group, head_dim, causal;
    uint32_t magic;       // r / group = (r * magic) >> shift for r < 2^31
    int32_t shift;
    float scale, scale2;  // scale, scale * log2(e)
};

__device__ __forceinline__ uint32_t div_group(const AttnParams &a, uint32_t r) {
    return (uint32_t)(((uint64_t)r * a.magic) >> a.shift);
}

// ------------------------------------------------------------------ LDS tiles
// A tile holds rows of DP elements (DP * sizeof(T) = 128, 256 or 512 bytes) in 16-byte
// chunks. ds_read_b128 serves lanes {0-7, 24-31}, {8-15, 16-23}, ... in one pass each over
// 16 units, and the fragment reads take 32 rows at one chunk; the transposing reads take
// four consecutive rows at four chunks. XORing the chunk with the row's low four bits, its
// two pairs exchanged, makes both conflict-free; 128-byte rows share a 256-byte line in
// pairs and use the line number the same way.
template <typename T, int DP>
struct Tile {
    static constexpr int kBytes = DP * (int)sizeof(T);
    static constexpr int kChunks = kBytes / 16;
    static constexpr int kFrags = kChunks / 2;   // 16-byte fragments of a row per lane half
    __device__ static __forceinline__ int addr(int r, int c) {
        if constexpr (kBytes == 128) {
            const int line = r >> 1;
            return line * 256 + (((((r & 1) << 3) | c) ^ (((line & 1) << 2) | ((line >> 1) & 3))) << 4);
        } else {
            return r * kBytes + ((c ^ (((r & 3) << 2) | ((r >> 2) & 3))) << 4);
        }
    }
};

typedef const __attribute__((address_space(3))) char lds_char;

__device__ __forceinline__ uint32_t lds_of(const void *p) { return (uint32_t)(uintptr_t)(lds_char *)p; }

__device__ __forceinline__ uint4 lds_read16(uint32_t at) {
    return __builtin_bit_cast(uint4, *(const __attribute__((address_space(3))) u32x4 *)(uintptr_t)at);
}
__device__ __forceinline__ uint2 lds_read_transposed(uint32_t at) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_kt_v4s *)(uintptr_t)at));
}

// A lane's byte offsets in a tile: of the chunks it reads as rows, and of those it reads
// transposed. `refresh` once a step keeps the sums with a stage's constant address out of
// registers: they become immediate offsets of the reads.
template <typename T, int DP>
struct Lanes {
    static constexpr int kFrags = Tile<T, DP>::kFrags, kCols = sizeof(T) == 2 ? DP / 16 : 1;
    uint32_t row[kFrags], col[kCols];
    __device__ __forceinline__ explicit Lanes(int lane) {
        const int h = lane >> 5;
#pragma unroll
        for (int s = 0; s < kFrags; ++s) row[s] = (uint32_t)Tile<T, DP>::addr(lane & 31, 2 * s + h);
        if constexpr (sizeof(T) == 2) {
            const int r = 4 * h + ((lane & 15) >> 2);
#pragma unroll
            for (int n = 0; n < DP / 32; ++n) {
                const int c = 4 * n + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), o = (lane & 1) * 8;
                col[2 * n] = (uint32_t)(Tile<T, DP>::addr(r, c) + o);
                col[2 * n + 1] = (uint32_t)(Tile<T, DP>::addr(r + 8, c) + o);
            }
        } else {
            col[0] = (uint32_t)lane;
        }
    }
    uint32_t moved = 0;   // float32: of the transposed reads
    // Reads from so many bytes further on.
    __device__ __forceinline__ void shift(uint32_t rows, uint32_t transposed) {
#pragma unroll
        for (int s = 0; s < kFrags; ++s) row[s] += rows;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int n = 0; n < kCols; ++n) col[n] += transposed;
        } else {
            moved = transposed;
        }
    }
    __device__ __forceinline__ void refresh() {
#pragma unroll
        for (int s = 0; s < kFrags; ++s) asm volatile("" : "+v"(row[s]));
#pragma unroll
        for (int n = 0; n < kCols; ++n) asm volatile("" : "+v"(col[n]));
    }
};

// acc[row, col] += sum_d tile[row0 + row][d] * frag[col][d]
template <typename T, int DP>
__device__ __forceinline__ void scores(f32x16 &acc, uint32_t tile, int row0, const uint4 (&frag)[Tile<T, DP>::kFrags],
                                       const Lanes<T, DP> &at) {
    const uint32_t base = tile + row0 * Tile<T, DP>::kBytes;
#pragma unroll
    for (int s = 0; s < Tile<T, DP>::kFrags; ++s) {
        const uint4 a = lds_read16(at.row[s] + base);
        if constexpr (sizeof(T) == 2) {
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                          __builtin_bit_cast(bf16x8, frag[s]), acc, 0, 0, 0);
        } else {
            const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, frag[s]);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], acc, 0, 0, 0);
        }
    }
}

// sum + the two values of a pair rounded to bf16 (v_dot2_f32_bf16).
__device__ __forceinline__ float add_pair(uint32_t pair, float sum) {
    const bf16x2_v ones = {(__bf16)1.0f, (__bf16)1.0f};
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_v, pair), ones, sum, false);
}

// acc[b][d, col] += sum_row tile[row0 + row][32 b + d] * p[row, col], p as `scores` leaves it:
// register i of lane half h is row 8 (i / 4) + 4 h + i % 4. `taken`: the sum of the lane's p as
// they enter the product.
template <typename T, int DP>
__device__ __forceinline__ void outer(f32x16 (&acc)[DP / 32], uint32_t tile, int row0, const f32x16 &p,
                                      const Lanes<T, DP> &at, float *taken = nullptr) {
    const uint32_t base = tile + row0 * Tile<T, DP>::kBytes;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            uint4 b;
            b.x = pack_bf16x2(p[8 * s], p[8 * s + 1]);
            b.y = pack_bf16x2(p[8 * s + 2], p[8 * s + 3]);
            b.z = pack_bf16x2(p[8 * s + 4], p[8 * s + 5]);
            b.w = pack_bf16x2(p[8 * s + 6], p[8 * s + 7]);
            if (taken) *taken = add_pair(b.w, add_pair(b.z, add_pair(b.y, add_pair(b.x, *taken))));
#pragma unroll
            for (int n = 0; n < DP / 32; ++n) {
                const uint2 l2 = lds_read_transposed(at.col[2 * n] + base + 16 * s * Tile<T, DP>::kBytes);
                const uint2 h2 = lds_read_transposed(at.col[2 * n + 1] + base + 16 * s * Tile<T, DP>::kBytes);
                const uint4 a = make_uint4(l2.x, l2.y, h2.x, h2.y);
                acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                                 __builtin_bit_cast(bf16x8, b), acc[n], 0, 0, 0);
            }
        }
    } else {
        const int lane = (int)at.col[0], h = lane >> 5;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = 8 * (i >> 2) + 4 * h + (i & 3);
#pragma unroll
            for (int n = 0; n < DP / 32; ++n) {
                const float a = *(const __attribute__((address_space(3))) float *)(uintptr_t)(
                    base + at.moved + Tile<T, DP>::addr(row, 8 * n + ((lane & 31) >> 2)) + (lane & 3) * 4);
                acc[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[i], acc[n], 0, 0, 0);
            }
        }
    }
}

// ------------------------------------------------------------------ global -> LDS
// One thread's share of a tile of ROWS rows, held in registers between the load and the
// LDS store. Rows that `valid` refuses are loaded from an offset past the buffer's range,
// which reads zeros: nothing behind a record's end enters a product (a masked zero times a NaN
// there would be NaN).
template <typename T, int DP, int ROWS, int THREADS>
struct Stage {
    static constexpr int kChunks = Tile<T, DP>::kChunks;
    static constexpr int kLoads = (ROWS * kChunks + THREADS - 1) / THREADS;
    static_assert(ROWS * kChunks % THREADS == 0 || kLoads == 1, "whole loads");
    static constexpr bool kPart = ROWS * kChunks < THREADS;   // some threads have none
    uint4 r[kLoads];
    __device__ static __forceinline__ int row_of(int p) { return (p * THREADS + (int)threadIdx.x) / kChunks; }
    __device__ static __forceinline__ int chunk_of() { return (int)threadIdx.x % kChunks; }   // THREADS % kChunks == 0
    // offset(p): bytes from base to the row of load p; valid(row): whether it exists.
    template <typename Offset, typename Valid>
    __device__ __forceinline__ void load(const char *base, int chunks, Offset offset, Valid valid) {
        const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(base, 0x7fffffff);
        const bool wanted = chunk_of() < chunks;
#pragma unroll
        for (int p = 0; p < kLoads; ++p) {
            const bool ok = wanted & valid(row_of(p)) & (!kPart || row_of(p) < ROWS);
            r[p] = buf_load16(rsrc, ok ? offset(p) + 16u * (uint32_t)chunk_of() : kOOB);
        }
    }
    __device__ __forceinline__ void store(uint4 *tile) const {
#pragma unroll
        for (int p = 0; p < kLoads; ++p)
            if (!kPart || row_of(p) < ROWS)
                *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(tile) + Tile<T, DP>::addr(row_of(p), chunk_of())) =
                    r[p];
    }
};

// A row's fragments as the B operand holds them: chunks 2 s + h of the row at `p`.
template <typename T, int DP>
__device__ __forceinline__ void row_fragments(const char *p, uint4 (&frag)[Tile<T, DP>::kFrags], bool valid,
                                              int chunks, int lane) {
#pragma unroll
    for (int s = 0; s < Tile<T, DP>::kFrags; ++s) {
        const int c = 2 * s + (lane >> 5);
        frag[s] = valid && c < chunks ? *reinterpret_cast<const uint4 *>(p + 16 * c) : zero4();
    }
}

__device__ __forceinline__ f32x16 splat(float v) {
    f32x16 r;
#pragma unroll
    for (int i = 0; i < 16; ++i) r[i] = v;
    return r;
}

// The wave's number in its workgroup, known to be the same in all its lanes.
__device__ __forceinline__ int wave_index() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// The lane, as a value that the compiler cannot carry from one piece of work to the next: what
// depends on it is made anew instead of filling registers through the main loop.
__device__ __forceinline__ int fresh_lane() {
    int lane = (int)threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

// Value of the same column in the other half of the wave.
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

// Four consecutive elements of a row at element d.
template <typename T>
__device__ __forceinline__ void store4(char *row, int d, float x, float y, float z, float w) {
    if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2 *>(row + 2 * d) = make_uint2(pack_bf16x2(x, y), pack_bf16x2(z, w));
    else
        *reinterpret_cast<float4 *>(row + 4 * d) = make_float4(x, y, z, w);
}
// What that rounding left of them.
template <typename T>
__device__ __forceinline__ void store4_rest(char *row, int d, float x, float y, float z, float w) {
    if constexpr (sizeof(T) == 2)
        store4<T>(row, d, x - bf16_to_f32(bf16_bits(x)), y - bf16_to_f32(bf16_bits(y)), z - bf16_to_f32(bf16_bits(z)),
                  w - bf16_to_f32(bf16_bits(w)));
}

// ------------------------------------------------------------------ rows of a forward or dq tile
struct RowOf {
    bool valid;
    int64_t token;    // in the whole tensor
    int head;
    int limit;        // keys the row sees
    __device__ __forceinline__ RowOf(const AttnParams &a, const Record &rec, int kv_head, int64_t r) {
        valid = r < rec.q_len * a.group;
        const uint32_t t = valid ? div_group(a, (uint32_t)r) : 0;
        token = rec.q_start + t;
        head = kv_head * a.group + (valid ? (int)((uint32_t)r - t * (uint32_t)a.group) : 0);
        const int64_t seen = a.causal ? (int64_t)t + 1 + rec.k_len - rec.q_len : rec.k_len;
        limit = seen < 0 ? 0 : (int)(seen < rec.k_len ? seen : rec.k_len);
    }
};

// Smallest and largest `limit` over the wave's valid rows (INT_MAX and 0 without any).
__device__ __forceinline__ void wave_limits(const RowOf &row, int &least, int &most) {
    least = row.valid ? row.limit : 0x7fffffff;
    most = row.valid ? row.limit : 0;
#pragma unroll
    for (int m = 16; m; m >>= 1) {
        least = min(least, __shfl_xor(least, m, 64));
        most = max(most, __shfl_xor(most, m, 64));
    }
    least = __builtin_amdgcn_readfirstlane(least);
    most = __builtin_amdgcn_readfirstlane(most);
}

// ------------------------------------------------------------------ the main loops
// dq runs over 32-key steps and dk/dv over 32-row steps in one rhythm: step t multiplies with
// tile t (the second products) while it makes the scores of tile t + 1, so that a wave always
// has matrix instructions beside its exponentials; tile t + 2 goes from registers to LDS and
// tile t + 3 from memory to registers. Three LDS stages, one barrier a step. The forward, which
// has no registers for a second set of scores, runs over tiles of kKeyTile keys in two stages: a
// tile's scores, its exponentials, its products, while the next one comes in.
constexpr int kStep = 32, kStages = 3;

// Runs f(stage, next, then) over consecutive steps with the stages as constants, so that LDS
// addresses are one register per lane pattern and immediate offsets.
template <typename F>
__device__ __forceinline__ void by_stage(int from, int to, F f) {
    typedef std::integral_constant<int, 0> Zero;
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 2> Two;
    for (int at = from; at < to; at += 3 * kStep) {
        f(at, Zero(), One(), Two());
        if (at + kStep < to) f(at + kStep, One(), Two(), Zero());
        if (at + 2 * kStep < to) f(at + 2 * kStep, Two(), Zero(), One());
    }
}

// Exponents scale2 (s - m) are one fused multiply-add of s with a rounded scale2 m, or in the
// backward with scale2 m + log2 of the sum. Past this size of scale2 m the rounding would show:
// p a factor of up to 2^(2^-24 scale2 m) off in the backward, and from 2^31 on p out of float32's
// range everywhere. Such rows' scores have m subtracted first, which is exact near m; for all
// rows that would cost 3% of the forward (632 us instead of 610 at 8192 rows of 32 heads).
constexpr float kFar = 64.0f;

__device__ __forceinline__ bool is_far(float m, float scale2) { return fabsf(m * scale2) > kFar; }

// Running softmax of a wave's 32 rows over their keys; m is the score that p and the sums are
// relative to, p = 2^(scale2 (s - m)).
struct Running {
    float m = -INFINITY, sum = 0.0f, taken = 0.0f;   // taken: the sum of p as rounded for the product
};

// What the backward needs of a row, apart: their sum would lose the logarithm where m is large.
__device__ __forceinline__ float2 row_stats(float m, float sum) {
    return sum == 0.0f ? make_float2(0.0f, INFINITY) : make_float2(m, __builtin_amdgcn_logf(sum));
}

// ------------------------------------------------------------------ forward
template <typename T>
constexpr int kKeyTile = sizeof(T) == 2 ? 64 : 32;

template <typename T, int DP>
__global__ __launch_bounds__(64 * kRowWaves, sizeof(T) == 2 || DP == 64 ? 2 : 1) void attention_forward(AttnParams a) {
    constexpr int KT = kKeyTile<T>, kUnits = KT * Tile<T, DP>::kChunks;
    __shared__ uint4 sk[2][kUnits], sv[2][kUnits];
    const Group group = a.groups[blockIdx.x / a.kv_heads];
    const int kv_head = blockIdx.x % a.kv_heads;
    for (int piece = 0; piece < group.count; ++piece) {
        const Item item = a.items[group.first + piece];
        const Record rec = a.records[item.record];
        const int lane = fresh_lane(), wave = wave_index(), chunks = a.head_dim * (int)sizeof(T) / 16;

        const RowOf row(a, rec, kv_head, (int64_t)item.begin + wave * kWaveCols + (lane & 31));
        int least, most;
        wave_limits(row, least, most);
        uint4 qf[Tile<T, DP>::kFrags];
        row_fragments<T, DP>(a.q + row.token * a.q_token + row.head * a.q_head, qf, row.valid, chunks, lane);

        const char *k0 = a.k + rec.k_start * a.k_token + kv_head * a.k_head;
        const char *v0 = a.v + rec.k_start * a.v_token + kv_head * a.v_head;
        Stage<T, DP, KT, 64 * kRowWaves> ks, vs;
        auto load = [&](int key) {
            const int left = (int)rec.k_len - key;
            auto valid = [&](int r) { return r < left; };
            ks.load(k0 + key * a.k_token, chunks,
                    [&](int p) { return (uint32_t)ks.row_of(p) * (uint32_t)a.k_token; }, valid);
            vs.load(v0 + key * a.v_token, chunks,
                    [&](int p) { return (uint32_t)vs.row_of(p) * (uint32_t)a.v_token; }, valid);
        };

        f32x16 o[DP / 32];
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) o[n] = splat(0.0f);
        Running run;
        if (item.lo < item.hi) {
            load(item.lo);
            ks.store(sk[0]);
            vs.store(sv[0]);
        }
        __syncthreads();
        Lanes<T, DP> at(lane);
        auto step = [&](int key, auto stage) {
            constexpr int buf = decltype(stage)::value;
            at.refresh();
            const bool more = key + KT < item.hi;
            if (more) load(key + KT);
            if (key < most) {
                f32x16 s[KT / 32];
#pragma unroll
                for (int t = 0; t < KT / 32; ++t) {
                    s[t] = splat(0.0f);
                    scores<T, DP>(s[t], lds_of(sk) + buf * (uint32_t)sizeof(sk[0]), 32 * t, qf, at);
                }
                if (key + KT > least) {
                    const int left = row.limit - key - 4 * (lane >> 5);
#pragma unroll
                    for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            s[t][i] = 32 * t + 8 * (i >> 2) + (i & 3) < left ? s[t][i] : -INFINITY;
                }
                float top = s[0][0];
#pragma unroll
                for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) top = fmaxf(top, s[t][i]);
                top = fmaxf(top, other_half(top));
                // The reference moves only when a row's maximum has grown by more than 2^8: p then
                // stays below 2^8, o and the sum are exact in that scale, and most tiles skip the
                // rescaling of o.
                if (__any((top - run.m) * a.scale2 > 8.0f)) {
                    const float grown = fmaxf(run.m, top);
                    const float shrink = grown == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f((run.m - grown) * a.scale2);
                    run.m = grown;
                    run.sum *= shrink;
                    run.taken *= shrink;
#pragma unroll
                    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[n][i] *= shrink;
                }
                const float m = run.m == -INFINITY ? 0.0f : run.m;
                float ref = m * a.scale2;
                if (__any(is_far(m, a.scale2))) {
                    ref = 0.0f;
#pragma unroll
                    for (int t = 0; t < KT / 32; ++t)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[t][i] -= m;
                }
#pragma unroll
                for (int t = 0; t < KT / 32; ++t) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][i], a.scale2, -ref));
                        run.sum += s[t][i];
                    }
                    outer<T, DP>(o, lds_of(sv) + buf * (uint32_t)sizeof(sv[0]), 32 * t, s[t], at, &run.taken);
                }
            }
            if (more) {
                ks.store(sk[buf ^ 1]);
                vs.store(sv[buf ^ 1]);
            }
            __syncthreads();
        };
        for (int key = item.lo; key < item.hi; key += 2 * KT) {
            step(key, std::integral_constant<int, 0>());
            if (key + KT < item.hi) step(key + KT, std::integral_constant<int, 1>());
        }

        const float sum = run.sum + other_half(run.sum);
        const float taken = sizeof(T) == 2 ? run.taken + other_half(run.taken) : sum;
        const int d0 = 4 * (lane >> 5);
        if (!row.valid) continue;
        if (item.slot < 0) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / taken;
            const int64_t at = row.token * a.o_token + row.head * a.o_head;
            char *dst = a.dst0 + at;
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int d = 32 * n + 2 * i + d0;
                    if (d >= a.head_dim) continue;
                    const float x = o[n][i] * inv, y = o[n][i + 1] * inv, z = o[n][i + 2] * inv, w = o[n][i + 3] * inv;
                    store4<T>(dst, d, x, y, z, w);
                    if (a.rest) store4_rest<T>(a.rest + at, d, x, y, z, w);
                }
            if (a.stats && lane < 32)
                a.stats[row.token * a.heads + row.head] = row_stats(run.m, sum);
        } else {
            const int64_t at = ((int64_t)item.slot * a.kv_heads + kv_head) * kRowTile + wave * kWaveCols + (lane & 31);
            float *dst = a.part0 + at * DP;
            const float scale = sum == 0.0f ? 0.0f : sum / taken;   // joined with the exact sums as weights
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4 *>(dst + 32 * n + 2 * i + d0) =
                        make_float4(o[n][i] * scale, o[n][i + 1] * scale, o[n][i + 2] * scale, o[n][i + 3] * scale);
            if (lane < 32) *reinterpret_cast<float2 *>(a.part1 + 2 * at) = make_float2(run.m, sum);
        }
    }
}

// Joins the key ranges of split rows: with M = max_s m_s, o = sum_s 2^(m_s - M) o_s over
// sum_s 2^(m_s - M) sum_s. DP / 4 threads per row and part; parts past the fourth of a row are
// shared out over up to 8 such teams, whose sums are added in order.
__host__ __device__ __forceinline__ int join_teams(int parts) {
    return parts <= 4 ? 1 : parts <= 8 ? 2 : parts <= 16 ? 4 : 8;
}
__host__ __device__ __forceinline__ int join_rows(int parts, int dp) { return kThreads / (dp / 4) / join_teams(parts); }

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void attention_join(AttnParams a, const Item *joins, int tile) {
    constexpr int kLanes = DP / 4;
    __shared__ float4 steams[kThreads];
    __shared__ float ssum[kThreads / kLanes];
    const Item join = joins[blockIdx.x / a.kv_heads];
    const int kv_head = blockIdx.x % a.kv_heads, teams = join_teams(join.hi);
    const int place = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, team = place % teams;
    const int r = join.slot + place / teams;
    const bool wanted = r < join.slot + join.rows;
    const int64_t first = ((int64_t)join.lo * a.kv_heads + kv_head) * tile + (wanted ? r : 0);
    const int64_t step = (int64_t)a.kv_heads * tile;
    float top = -INFINITY;
#pragma unroll 4
    for (int s = 0; s < join.hi; ++s) top = fmaxf(top, a.part1[2 * (first + s * step)]);
    const float ref = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int s = team; s < join.hi; s += teams) {
        const int64_t at = first + s * step;
        const float2 ms = *reinterpret_cast<const float2 *>(a.part1 + 2 * at);
        const float4 x = *reinterpret_cast<const float4 *>(a.part0 + at * DP + 4 * lane);
        const float w = __builtin_amdgcn_exp2f((ms.x - ref) * a.scale2);
        sum = __builtin_fmaf(w, ms.y, sum);
        acc.x = __builtin_fmaf(w, x.x, acc.x);
        acc.y = __builtin_fmaf(w, x.y, acc.y);
        acc.z = __builtin_fmaf(w, x.z, acc.z);
        acc.w = __builtin_fmaf(w, x.w, acc.w);
    }
    if (teams > 1) {
        steams[threadIdx.x] = acc;
        if (lane == 0) ssum[place] = sum;
        __syncthreads();
        if (team) return;
        for (int t = 1; t < teams; ++t) {
            const float4 x = steams[threadIdx.x + t * kLanes];
            sum += ssum[place + t];
            acc.x += x.x;
            acc.y += x.y;
            acc.z += x.z;
            acc.w += x.w;
        }
    }
    if (!wanted) return;
    const Record rec = a.records[join.record];
    const RowOf row(a, rec, kv_head, (int64_t)join.begin + r);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t at = row.token * a.o_token + row.head * a.o_head;
    acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    if (4 * lane < a.head_dim) {
        store4<T>(a.dst0 + at, 4 * lane, acc.x, acc.y, acc.z, acc.w);
        if (a.rest) store4_rest<T>(a.rest + at, 4 * lane, acc.x, acc.y, acc.z, acc.w);
    }
    if (a.stats && lane == 0)
        a.stats[row.token * a.heads + row.head] = row_stats(top, sum);
}

// Sum of the parts of one row or key, in order, for four elements.
template <int DP>
__device__ __forceinline__ float4 sum_parts(const float *part, int64_t at, int64_t step, int count) {
    float4 v = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int s = 0; s < count; ++s) {
        const float4 x = *reinterpret_cast<const float4 *>(part + (at + s * step) * DP);
        v.x += x.x;
        v.y += x.y;
        v.z += x.z;
        v.w += x.w;
    }
    return v;
}

// ------------------------------------------------------------------ dq (and the rows' terms)
template <typename T>
__device__ __forceinline__ float dot_chunk(const uint4 &x, const uint4 &y, float acc) {
    const uint32_t p[4] = {x.x, x.y, x.z, x.w}, q[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 2) {
            acc = __builtin_fmaf(__builtin_bit_cast(float, p[j] << 16), __builtin_bit_cast(float, q[j] << 16), acc);
            acc = __builtin_fmaf(__builtin_bit_cast(float, p[j] & 0xffff0000u),
                                 __builtin_bit_cast(float, q[j] & 0xffff0000u), acc);
        } else {
            acc = __builtin_fmaf(__builtin_bit_cast(float, p[j]), __builtin_bit_cast(float, q[j]), acc);
        }
    }
    return acc;
}

template <typename T, int DP>
__global__ __launch_bounds__(64 * kRowWaves, sizeof(T) == 2 || DP == 64 ? 2 : 1) void attention_dq(AttnParams a) {
    constexpr int kUnits = kStep * Tile<T, DP>::kChunks;
    __shared__ uint4 sk[kStages][kUnits], sv[kStages][kUnits];
    const Group group = a.groups[blockIdx.x / a.kv_heads];
    const int kv_head = blockIdx.x % a.kv_heads;
    for (int piece = 0; piece < group.count; ++piece) {
        const Item item = a.items[group.first + piece];
        const Record rec = a.records[item.record];
        const int lane = fresh_lane(), wave = wave_index(), chunks = a.head_dim * (int)sizeof(T) / 16;

        const RowOf row(a, rec, kv_head, (int64_t)item.begin + wave * kWaveCols + (lane & 31));
        int least, most;
        wave_limits(row, least, most);
        most = min(most, item.hi);
        uint4 qf[Tile<T, DP>::kFrags], gf[Tile<T, DP>::kFrags];
        row_fragments<T, DP>(a.dout + row.token * a.do_token + row.head * a.do_head, gf, row.valid, chunks, lane);
        row_fragments<T, DP>(a.out + row.token * a.o_token + row.head * a.o_head, qf, row.valid, chunks, lane);
        float delta = 0.0f;
#pragma unroll
        for (int s = 0; s < Tile<T, DP>::kFrags; ++s) delta = dot_chunk<T>(gf[s], qf[s], delta);
        if (sizeof(T) == 2 && a.rest) {
            row_fragments<T, DP>(a.rest + row.token * a.o_token + row.head * a.o_head, qf, row.valid, chunks, lane);
#pragma unroll
            for (int s = 0; s < Tile<T, DP>::kFrags; ++s) delta = dot_chunk<T>(gf[s], qf[s], delta);
        }
        delta += other_half(delta);
        float m = 0.0f, lse = INFINITY;
        if (row.valid) {
            const int64_t at = row.token * a.heads + row.head;
            const float2 stats = a.stats[at];
            m = stats.x;
            lse = stats.y;
        }
        if (row.valid && lane < 32 && item.lo == 0) {
            const bool far = is_far(m, a.scale2);
            a.terms[row.token * a.heads + row.head] =
                make_float4(far ? m : 0.0f, far ? -lse : -__builtin_fmaf(m, a.scale2, lse), -delta, far ? 1.0f : 0.0f);
        }
        const bool far = __any(is_far(m, a.scale2));
        if (!far) lse = __builtin_fmaf(m, a.scale2, lse);
        row_fragments<T, DP>(a.q + row.token * a.q_token + row.head * a.q_head, qf, row.valid, chunks, lane);

        const char *k0 = a.k + rec.k_start * a.k_token + kv_head * a.k_head;
        const char *v0 = a.v + rec.k_start * a.v_token + kv_head * a.v_head;
        Stage<T, DP, kStep, 64 * kRowWaves> ks, vs;
        auto load = [&](int key) {
            const int left = (int)rec.k_len - key;
            auto valid = [&](int r) { return r < left; };
            ks.load(k0 + key * a.k_token, chunks,
                    [&](int p) { return (uint32_t)ks.row_of(p) * (uint32_t)a.k_token; }, valid);
            vs.load(v0 + key * a.v_token, chunks,
                    [&](int p) { return (uint32_t)vs.row_of(p) * (uint32_t)a.v_token; }, valid);
        };
        auto store = [&](int buf) {
            ks.store(sk[buf]);
            vs.store(sv[buf]);
        };

        f32x16 o[DP / 32], s, g;
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) o[n] = splat(0.0f);
        if (item.lo < item.hi) {
            load(item.lo);
            store(0);
            if (item.lo + kStep < item.hi) {
                load(item.lo + kStep);
                store(1);
                if (item.lo + 2 * kStep < item.hi) load(item.lo + 2 * kStep);
            }
        }
        __syncthreads();
        Lanes<T, DP> at(lane);
        auto both = [&](int buf) {
            s = splat(0.0f);
            g = splat(-delta);
            scores<T, DP>(s, lds_of(sk) + buf * (uint32_t)sizeof(sk[0]), 0, qf, at);
            scores<T, DP>(g, lds_of(sv) + buf * (uint32_t)sizeof(sv[0]), 0, gf, at);
        };
        if (item.lo < most) both(0);
        by_stage(item.lo, item.hi, [&](int key, auto now_, auto next_, auto then_) {
            constexpr int now = decltype(now_)::value, next = decltype(next_)::value, then = decltype(then_)::value;
            if (key + 2 * kStep < item.hi) {
                store(then);
                if (key + 3 * kStep < item.hi) load(key + 3 * kStep);
            }
            if (key < most) {
                at.refresh();
                if (far) {
                    const float m = row.valid ? a.stats[row.token * a.heads + row.head].x : 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] -= m;
                }
                f32x16 ds;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    ds[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale2, -lse)) * g[i];
                if (key + kStep > least) {
                    const int left = row.limit - key - 4 * (lane >> 5);
#pragma unroll
                    for (int i = 0; i < 16; ++i) ds[i] = 8 * (i >> 2) + (i & 3) < left ? ds[i] : 0.0f;
                }
                if (key + kStep < most) both(next);
                outer<T, DP>(o, lds_of(sk) + now * (uint32_t)sizeof(sk[0]), 0, ds, at);
            }
            __syncthreads();
        });
        if (!row.valid) continue;
        const int d0 = 4 * (lane >> 5);
        if (item.slot < 0) {
            char *dst = a.dst0 + row.token * a.d_token + (int64_t)row.head * a.head_dim * (int)sizeof(T);
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int d = 32 * n + 2 * i + d0;
                    if (d < a.head_dim)
                        store4<T>(dst, d, o[n][i] * a.scale, o[n][i + 1] * a.scale, o[n][i + 2] * a.scale,
                                  o[n][i + 3] * a.scale);
                }
        } else {
            float *dst = a.part0 + (((int64_t)item.slot * a.kv_heads + kv_head) * kRowTile + wave * kWaveCols +
                                    (lane & 31)) * DP;
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4 *>(dst + 32 * n + 2 * i + d0) =
                        make_float4(o[n][i], o[n][i + 1], o[n][i + 2], o[n][i + 3]);
        }
    }
}

template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void attention_dq_join(AttnParams a, const Item *joins, int tile) {
    const Item join = joins[blockIdx.x / a.kv_heads];
    const int kv_head = blockIdx.x % a.kv_heads, place = threadIdx.x / (DP / 4), d = threadIdx.x % (DP / 4) * 4;
    if (place >= join.rows || d >= a.head_dim) return;
    const int64_t step = (int64_t)a.kv_heads * tile;
    const float4 v = sum_parts<DP>(a.part0 + d, ((int64_t)join.lo * a.kv_heads + kv_head) * tile + join.slot + place, step,
                                   join.hi);
    const Record rec = a.records[join.record];
    const RowOf row(a, rec, kv_head, (int64_t)join.begin + join.slot + place);
    store4<T>(a.dst0 + row.token * a.d_token + (int64_t)row.head * a.head_dim * (int)sizeof(T), d, v.x * a.scale,
              v.y * a.scale, v.z * a.scale, v.w * a.scale);
}

// ------------------------------------------------------------------ dk, dv
// Two waves share 32 keys. One makes the probabilities p = exp(s - lse) and dv += p^T do, the
// other do . v - delta, ds = p (do . v - delta) with the first one's p through LDS (lane by
// lane: both hold the same layout) and dk += ds^T q. Each then holds one operand of keys and
// one accumulator, which leaves room for two waves per SIMD; a single wave with both needs
// 490 registers and ran at 25% of the matrix instructions' rate (2633 us at 8192 rows of 32
// heads, this form 1936 with the same shares of work, 1388 with even ones).
constexpr int kKeyWaves = 8;

template <typename T, int DP>
__global__ __launch_bounds__(64 * kKeyWaves, sizeof(T) == 2 && DP == 64 ? 4 : 2) void attention_dkv(AttnParams a) {
    constexpr int kUnits = kStep * Tile<T, DP>::kChunks, kAll = 64 * kKeyWaves;
    __shared__ uint4 st[2][kStages][kUnits];                     // q, dout
    __shared__ __align__(16) float sstat[3][kStages][kStep];   // m of far rows, -lse (far: -log2 sum), -delta
    __shared__ int sfar[kStages];                               // whether any row is far
    __shared__ __align__(16) float szero[kStep];
    __shared__ f32x4 sp[2][kKeyWaves / 2][4][64];
    const Group group = a.groups[blockIdx.x / a.kv_heads];
    const int kv_head = blockIdx.x % a.kv_heads;
    for (int piece = 0; piece < group.count; ++piece) {
        const Item item = a.items[group.first + piece];
        const Record rec = a.records[item.record];
        const int lane = fresh_lane(), wave = wave_index(), chunks = a.head_dim * (int)sizeof(T) / 16;
        const int pair = wave & 3;                // waves w and w + 4 run on one SIMD
        const bool for_dv = wave < kKeyWaves / 2;

        const int key0 = item.begin + pair * kWaveCols, key = key0 + (lane & 31);
        const bool valid = key < rec.k_len;
        const int64_t kv = rec.k_start + (valid ? key : 0);
        uint4 frag[Tile<T, DP>::kFrags];
        row_fragments<T, DP>(for_dv ? a.k + kv * a.k_token + kv_head * a.k_head : a.v + kv * a.v_token + kv_head * a.v_head,
                             frag, valid, chunks, lane);

        const int nrows = (int)(rec.q_len * a.group);
        // Row r sees key j when r >= first(j); tokens before key j - (keys - queries) do not.
        auto first = [&](int j) -> int64_t {
            const int64_t t = a.causal ? j - (rec.k_len - rec.q_len) : 0;
            return t < 0 ? 0 : t * a.group;
        };
        const int64_t mine = first(key), wave_first = first(key0), wave_last = first(key0 + kWaveCols - 1);

        Stage<T, DP, kStep, kAll> qs, gs;
        float4 stat_r = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        // A group that divides the step makes a row's token and head the same in every step; the
        // others are divided out each time.
        const bool regular = kStep % a.group == 0;
        const int stat_row = (int)threadIdx.x % kStep;
        struct Place {
            uint32_t q, g;
            int32_t stat;
        };
        auto place = [&](int row, uint32_t base) -> Place {   // row after the first token of the step
            const uint32_t r = base + (uint32_t)row, t = div_group(a, r), h = r - t * (uint32_t)a.group;
            return {t * (uint32_t)a.q_token + h * (uint32_t)a.q_head, t * (uint32_t)a.do_token + h * (uint32_t)a.do_head,
                    (int32_t)(t * (uint32_t)a.heads + h)};
        };
        constexpr int kLoads = Stage<T, DP, kStep, kAll>::kLoads;
        Place fixed[kLoads];
#pragma unroll
        for (int p = 0; p < kLoads; ++p) fixed[p] = place(qs.row_of(p), 0);
        const int32_t fixed_stat = place(stat_row, 0).stat;
        auto load = [&](int r0) {
            const uint32_t t0 = div_group(a, (uint32_t)r0), base = (uint32_t)r0 - t0 * (uint32_t)a.group;
            const int64_t token = rec.q_start + t0;
            const int left = nrows - r0;
            Place at[kLoads];
            int32_t stat = fixed_stat;
#pragma unroll
            for (int p = 0; p < kLoads; ++p) at[p] = fixed[p];
            if (!regular) {
#pragma unroll
                for (int p = 0; p < kLoads; ++p) at[p] = place(qs.row_of(p), base);
                stat = place(stat_row, base).stat;
            }
            auto exists = [&](int row) { return row < left; };
            qs.load(a.q + token * a.q_token + (int64_t)kv_head * a.group * a.q_head, chunks, [&](int p) { return at[p].q; },
                    exists);
            gs.load(a.dout + token * a.do_token + (int64_t)kv_head * a.group * a.do_head, chunks,
                    [&](int p) { return at[p].g; }, exists);
            if (wave == kKeyWaves / 2 && lane < kStep)   // rows behind the last: p = 0
                stat_r = stat_row < left ? a.terms[token * a.heads + kv_head * a.group + stat]
                                         : make_float4(0.0f, -INFINITY, 0.0f, 0.0f);
        };
        auto store = [&](int buf) {
            qs.store(st[0][buf]);
            gs.store(st[1][buf]);
            if (wave == kKeyWaves / 2) {
                const bool any = __any(stat_r.w != 0.0f);
                if (lane < kStep) {
                    sstat[0][buf][lane] = stat_r.x;
                    sstat[1][buf][lane] = stat_r.y;
                    sstat[2][buf][lane] = stat_r.z;
                }
                if (lane == 0) sfar[buf] = any;
            }
        };

        f32x16 acc[DP / 32], s = splat(0.0f);
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) acc[n] = splat(0.0f);
        // Both roles run the same reads, from places of their own: scores with q, from zero, and the
        // second product with dout, or the other way round and from -delta.
        constexpr uint32_t kOther = sizeof(st[0]), kStage = sizeof(st[0][0]), kStat = sizeof(sstat[0][0]);
        Lanes<T, DP> at(lane);
        at.shift(for_dv ? 0 : kOther, for_dv ? kOther : 0);
        const uint32_t start = 16 * (lane >> 5) + (for_dv ? lds_of(szero) : lds_of(sstat) + 2 * kStages * kStat);
        const uint32_t start_step = for_dv ? 0 : kStat, own_stat = lds_of(sstat) + 16 * (lane >> 5);
        if (threadIdx.x < kStep) szero[threadIdx.x] = 0.0f;
        // Probabilities (for dv, shared) or do . v - delta of the rows at r0 in stage `buf`.
        auto make = [&](int r0, int buf, int turn) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 v = __builtin_bit_cast(f32x4, lds_read16(start + buf * start_step + 32 * i));
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * i + e] = v[e];
            }
            scores<T, DP>(s, lds_of(st) + buf * kStage, 0, frag, at);
            if (for_dv) {
                if (__builtin_amdgcn_readfirstlane(sfar[buf])) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const f32x4 m = __builtin_bit_cast(f32x4, lds_read16(own_stat + buf * kStat + 32 * i));
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[4 * i + e] -= m[e];
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 v = __builtin_bit_cast(f32x4, lds_read16(own_stat + (kStages + buf) * kStat + 32 * i));
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s[4 * i + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i + e], a.scale2, v[e]));
                }
                if (r0 < wave_last) {
                    // rows below `hidden` do not see the key
                    const int hidden = (int)(mine < nrows ? mine : nrows) - r0 - 4 * (lane >> 5);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = 8 * (i >> 2) + (i & 3) >= hidden ? s[i] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sp[turn][pair][i][lane] = f32x4{s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]};
            }
        };
        if (item.lo < item.hi) {
            load(item.lo);
            store(0);
            if (item.lo + kStep < item.hi) {
                load(item.lo + kStep);
                store(1);
                if (item.lo + 2 * kStep < item.hi) load(item.lo + 2 * kStep);
            }
        }
        __syncthreads();
        int turn = 0;
        if (item.lo < item.hi && item.lo + kStep > wave_first) make(item.lo, 0, 0);
        __syncthreads();
        by_stage(item.lo, item.hi, [&](int r0, auto now_, auto next_, auto then_) {
            constexpr int now = decltype(now_)::value, next = decltype(next_)::value, then = decltype(then_)::value;
            if (r0 + 2 * kStep < item.hi) {
                store(then);
                if (r0 + 3 * kStep < item.hi) load(r0 + 3 * kStep);
            }
            at.refresh();
            const bool seen = r0 + kStep > wave_first, more = r0 + kStep < item.hi && r0 + 2 * kStep > wave_first;
            f32x16 z = s;
            if (seen && !for_dv) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4 p = sp[turn][pair][i][lane];
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[4 * i + e] *= p[e];
                }
                if (r0 < wave_last) {   // 0 x inf
                    const int hidden = (int)(mine < nrows ? mine : nrows) - r0 - 4 * (lane >> 5);
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[i] = 8 * (i >> 2) + (i & 3) >= hidden ? z[i] : 0.0f;
                }
            }
            if (more) make(r0 + kStep, next, turn ^ 1);
            if (seen) outer<T, DP>(acc, lds_of(st) + now * kStage, 0, z, at);
            __syncthreads();
            turn ^= 1;
        });
        const int d0 = 4 * (lane >> 5);
        const float scale = for_dv ? 1.0f : a.scale;
        if (item.slot < 0) {
            if (!valid) continue;
            char *dst = (for_dv ? a.dst1 : a.dst0) + kv * a.d_token + (int64_t)kv_head * a.head_dim * (int)sizeof(T);
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int d = 32 * n + 2 * i + d0;
                    if (d < a.head_dim)
                        store4<T>(dst, d, acc[n][i] * scale, acc[n][i + 1] * scale, acc[n][i + 2] * scale,
                                  acc[n][i + 3] * scale);
                }
        } else {
            float *dst = (for_dv ? a.part1 : a.part0) +
                         (((int64_t)item.slot * a.kv_heads + kv_head) * kTile + pair * kWaveCols + (lane & 31)) * DP;
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4 *>(dst + 32 * n + 2 * i + d0) =
                        make_float4(acc[n][i], acc[n][i + 1], acc[n][i + 2], acc[n][i + 3]);
        }
    }
}

// Sums the row ranges of split key tiles in order: one thread per four elements of a key.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void attention_dkv_join(AttnParams a, const Item *joins) {
    const Item join = joins[blockIdx.x / a.kv_heads];
    const int kv_head = blockIdx.x % a.kv_heads, place = threadIdx.x / (DP / 4), d = threadIdx.x % (DP / 4) * 4;
    if (place >= join.rows || d >= a.head_dim) return;
    const int64_t step = (int64_t)a.kv_heads * kTile;
    const int64_t at = ((int64_t)join.lo * a.kv_heads + kv_head) * kTile + join.slot + place;
    const float4 dk = sum_parts<DP>(a.part0 + d, at, step, join.hi), dv = sum_parts<DP>(a.part1 + d, at, step, join.hi);
    const int64_t key = a.records[join.record].k_start + join.begin + join.slot + place;
    const int64_t off = key * a.d_token + (int64_t)kv_head * a.head_dim * (int)sizeof(T);
    store4<T>(a.dst0 + off, d, dk.x * a.scale, dk.y * a.scale, dk.z * a.scale, dk.w * a.scale);
    store4<T>(a.dst1 + off, d, dv.x, dv.y, dv.z, dv.w);
}

// ------------------------------------------------------------------ host side
constexpr int64_t kMaxRows = 0x7fffffff - 2 * kTile;

// A piece's fixed cost (its rows' or keys' load, its result's store) in units of kUnit: the
// smaller it is, the more pieces and partials there are. Measured, three records of 3421 tokens of
// 16 heads, forward: 53 us with kRowFixed = 1, 43 with 3, 40 with 6, which takes 51 instead of 50 at
// 24 tokens of one row. kKeyFixed = 3, 6 and 12: the same within 1%. Two float32 records of 833 rows
// of 8 heads, forward and backward: 85 us with kF32Fixed = 1, 111 with 3, 176 with 6; its few rows
// are short of workgroups, not of joins.
constexpr int64_t kRowFixed = 3, kKeyFixed = 6, kF32Fixed = 1;
constexpr int64_t kMaxPitch = (int64_t)1 << 24;   // bytes between tokens of k and v

// 64 packed rows span at most 64 / group + 2 tokens and all heads of the group.
bool row_span_ok(int64_t token, int64_t head, int64_t group) {
    return (64 / group + 2) * (double)token + (double)group * (double)head < 2147483647.0 - 1024;
}

int padded_dim(int64_t head_dim) { return head_dim <= 64 ? 64 : 128; }

bool dims_ok(int64_t heads, int64_t kv_heads, int64_t head_dim) {
    return heads > 0 && kv_heads > 0 && heads <= 65536 && heads % kv_heads == 0 && head_dim >= 8 && head_dim <= 128 &&
           head_dim % 8 == 0;
}

int fill_params(const ct_attention *c, AttnParams &a) {
    if (!c) return -CT_EINVAL_POINTER;
    if (c->dtype != CT_BF16 && c->dtype != CT_F32) return -CT_EINVAL_DTYPE;
    if (!dims_ok(c->heads, c->kv_heads, c->head_dim) || !(c->scale > 0.0f) || !(c->scale < INFINITY))
        return -CT_EINVAL_SHAPE;
    if (!c->q || !c->k || !c->v || !c->records) return -CT_EINVAL_POINTER;
    const int64_t size = c->dtype == CT_BF16 ? 2 : 4;
    const int64_t strides[6] = {c->q_token, c->q_head, c->k_token, c->k_head, c->v_token, c->v_head};
    for (int64_t s : strides)
        if (s < 0 || s * size % 16 || s > (int64_t)1 << 40) return -CT_EINVAL_SHAPE;
    if (((uintptr_t)c->q | (uintptr_t)c->k | (uintptr_t)c->v) % 16) return -CT_EINVAL_POINTER;
    a = AttnParams{};
    a.q = (const char *)c->q;
    a.k = (const char *)c->k;
    a.v = (const char *)c->v;
    a.q_token = c->q_token * size;
    a.q_head = c->q_head * size;
    a.k_token = c->k_token * size;
    a.k_head = c->k_head * size;
    a.v_token = c->v_token * size;
    a.v_head = c->v_head * size;
    a.o_head = c->head_dim * size;
    a.o_token = c->heads * a.o_head;
    a.records = (const Record *)c->records;
    a.heads = c->heads;
    a.kv_heads = c->kv_heads;
    a.group = c->heads / c->kv_heads;
    a.head_dim = c->head_dim;
    a.causal = c->causal ? 1 : 0;
    a.scale = c->scale;
    a.scale2 = c->scale * kLog2e;
    a.rest = c->dtype == CT_BF16 ? (char *)c->rest : nullptr;
    if ((uintptr_t)a.rest % 16) return -CT_EINVAL_POINTER;
    // r / group for r < 2^31: with 2^s >= group and M = floor(2^(31+s) / group) + 1,
    // r M / 2^(31+s) exceeds r / group by less than 1 / group.
    int s = 0;
    while ((1 << s) < a.group) ++s;
    a.magic = (uint32_t)(((uint64_t)1 << (31 + s)) / (uint64_t)a.group + 1);
    a.shift = 31 + s;
    // 32-bit offsets inside a tile: 64 rows of keys, and the tokens and heads of 64 packed rows.
    if (a.k_token > kMaxPitch || a.v_token > kMaxPitch) return -CT_EINVAL_SHAPE;
    if (!row_span_ok(a.q_token, a.q_head, a.group)) return -CT_EINVAL_SHAPE;
    return 0;
}

int status_of_last_launch() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : (int)e;
}

template <typename F>
int by_type(int dtype, int dp, F f) {
    typedef std::integral_constant<int, 64> Narrow;
    typedef std::integral_constant<int, 128> Wide;
    if (dtype == CT_BF16) return dp == 64 ? f((uint16_t)0, Narrow()) : f((uint16_t)0, Wide());
    return dp == 64 ? f(0.0f, Narrow()) : f(0.0f, Wide());
}

int64_t parts_per_item(int32_t pass, int dp) {   // floats
    return pass == CT_ATTENTION_KEYS ? 2 * (int64_t)kTile * dp
                                     : (int64_t)kRowTile * (dp + (pass == CT_ATTENTION_FORWARD ? 2 : 0));
}

// Workgroups that the card runs at once, by their registers: two of 4 waves per CU in the
// forward and dq (one for float32 with heads past 64), one of 8 waves in the dk, dv kernel (two
// for bf16 with heads up to 64).
int64_t groups_at_once(int32_t pass, int dp, int dtype) {
    if (pass == CT_ATTENTION_KEYS) return dp > 64 || dtype == CT_F32 ? 256 : 512;
    return dp > 64 && dtype == CT_F32 ? 256 : 512;
}

constexpr int64_t kUnit = 64;   // keys or rows: pieces are cut at its multiples

int64_t units_of(const Item &it) { return cdiv(it.hi - it.lo, kUnit); }

// Fills workgroups one after the other with the tiles' units until each has taken `cap`, where
// a piece costs its units and `fixed` (its rows' or keys' load, its result's store). Returns the
// number of workgroups; with `groups`, writes them and their pieces down.
int64_t fill(const std::vector<Item> &tiles, int64_t cap, int64_t fixed, std::vector<Item> *pieces,
             std::vector<Group> *groups) {
    int64_t count = 0, left = 0;
    for (const Item &tile : tiles) {
        for (int64_t lo = tile.lo;;) {
            const int64_t units = cdiv(tile.hi - lo, kUnit);
            // a workgroup's rest that is too short for its fixed cost stays unused
            if (left < fixed + std::min<int64_t>(units, fixed)) {
                left = cap;
                ++count;
                if (groups) groups->push_back({(int32_t)pieces->size(), 0, {}});
            }
            const int64_t take = std::min<int64_t>(units, std::max<int64_t>(1, left - fixed));
            left -= take + fixed;
            if (groups) {
                Item piece = tile;
                piece.lo = (int32_t)lo;
                piece.hi = (int32_t)std::min<int64_t>(tile.hi, lo + take * kUnit);
                piece.slot = piece.lo == tile.lo && piece.hi == tile.hi ? -1 : 0;
                pieces->push_back(piece);
                ++groups->back().count;
            }
            lo += take * kUnit;
            if (lo >= tile.hi) break;
        }
    }
    return count;
}

struct Plan {
    std::vector<Item> pieces, joins;
    std::vector<Group> groups;
    int64_t slots = 0;
};

void make_plan(int32_t pass, const Record *rec, int64_t n, int64_t kv_heads, int64_t group, int dp, bool causal, int dtype,
               Plan &plan) {
    const bool keys = pass == CT_ATTENTION_KEYS;
    const int64_t tile = keys ? kTile : kRowTile;
    std::vector<Item> tiles;
    int64_t work = 0, longest = 0;
    for (int64_t i = 0; i < n; ++i) {
        const int64_t rows = rec[i].q_len * group, shift = rec[i].k_len - rec[i].q_len;
        const int64_t span = keys ? rec[i].k_len : rows;
        for (int64_t b = 0; b < span; b += tile) {
            Item it = {};
            it.record = (int32_t)i;
            it.begin = (int32_t)b;
            it.slot = -1;
            it.rows = (int32_t)std::min(tile, span - b);
            if (keys) {   // rows that see the tile's first key, from a whole tile of rows on
                const int64_t t = causal ? std::max<int64_t>(0, b - shift) : 0;
                it.lo = (int32_t)std::min(t * group / kUnit * kUnit, rows);
                it.hi = (int32_t)rows;
            } else {      // keys that the tile's last row sees
                const int64_t t = (b + it.rows - 1) / group;
                it.hi = (int32_t)(causal ? std::min(rec[i].k_len, std::max<int64_t>(0, t + 1 + shift)) : rec[i].k_len);
            }
            work += units_of(it);
            longest = std::max(longest, units_of(it));
            tiles.push_back(it);
        }
    }
    const int64_t at_once = std::max<int64_t>(1, groups_at_once(pass, dp, dtype) / kv_heads);
    if ((int64_t)tiles.size() >= 2 * at_once && longest * at_once <= work) {
        // Enough whole tiles, none of them longer than a workgroup's share: longest first, so
        // that what starts last ends soon.
        std::stable_sort(tiles.begin(), tiles.end(),
                         [](const Item &x, const Item &y) { return units_of(x) > units_of(y); });
        for (const Item &it : tiles) {
            plan.groups.push_back({(int32_t)plan.pieces.size(), 1, {}});
            plan.pieces.push_back(it);
        }
        return;
    }
    // Otherwise every workgroup gets the same share of all units, cutting tiles where it ends.
    const int64_t fixed = dtype == CT_F32 ? kF32Fixed : keys ? kKeyFixed : kRowFixed;
    int64_t low = 2 * fixed, high = std::max<int64_t>(low, work + fixed * (int64_t)tiles.size());
    while (low < high) {
        const int64_t mid = (low + high) / 2;
        if (fill(tiles, mid, fixed, nullptr, nullptr) <= at_once) high = mid;
        else low = mid + 1;
    }
    fill(tiles, high, fixed, &plan.pieces, &plan.groups);
    for (size_t k = 0; k < plan.pieces.size();) {
        if (plan.pieces[k].slot < 0) {
            ++k;
            continue;
        }
        Item join = plan.pieces[k];
        join.lo = (int32_t)plan.slots;
        const size_t from = k;
        for (; k < plan.pieces.size() && plan.pieces[k].record == join.record && plan.pieces[k].begin == join.begin; ++k)
            plan.pieces[k].slot = (int32_t)plan.slots++;
        join.hi = (int32_t)(k - from);
        const int at_a_time = pass == CT_ATTENTION_FORWARD ? join_rows(join.hi, dp) : kThreads / (dp / 4);
        const int32_t rows = join.rows;
        for (int32_t r = 0; r < rows; r += at_a_time) {
            join.slot = r;
            join.rows = std::min(at_a_time, rows - r);
            plan.joins.push_back(join);
        }
    }
    // The pieces keep their order; the workgroups with most to do start first.
    auto cost = [&](const Group &g) {
        int64_t c = 0;
        for (int32_t k = 0; k < g.count; ++k) c += units_of(plan.pieces[(size_t)(g.first + k)]) + fixed;
        return c;
    };
    std::stable_sort(plan.groups.begin(), plan.groups.end(),
                     [&](const Group &x, const Group &y) { return cost(x) > cost(y); });
}

// counts: pieces, joins, partials, workgroups.
bool counts_ok(const int64_t *counts, int64_t kv_heads) {
    for (int i = 0; i < 4; ++i)
        if (counts[i] < 0 || counts[i] > 0x7fffffff / (kTile * kv_heads)) return false;
    return true;
}

void set_plan(AttnParams &a, const int32_t *plan, const int64_t *counts) {
    a.items = reinterpret_cast<const Item *>(plan);
    a.groups = reinterpret_cast<const Group *>(a.items + counts[0] + counts[1]);
}

}  // namespace
}  // namespace ct

using namespace ct;

static_assert(sizeof(Item) == 4 * kEntry && sizeof(Group) == 4 * kEntry, "plan entries");

extern "C" int ct_attention_plan(int32_t pass, const int64_t *records, int64_t n_records, int32_t heads,
                                 int32_t kv_heads, int32_t head_dim, int32_t dtype, int32_t causal,
                                 int32_t *entries, int64_t capacity, int64_t *counts) {
    if (pass < CT_ATTENTION_FORWARD || pass > CT_ATTENTION_KEYS || n_records < 0 || n_records > 0x7fffffff ||
        !dims_ok(heads, kv_heads, head_dim))
        return -CT_EINVAL_SHAPE;
    if (dtype != CT_BF16 && dtype != CT_F32) return -CT_EINVAL_DTYPE;
    if (!counts || (n_records && !records)) return -CT_EINVAL_POINTER;
    const int64_t group = heads / kv_heads;
    const Record *rec = reinterpret_cast<const Record *>(records);
    int64_t tiles = 0;
    for (int64_t i = 0; i < n_records; ++i) {
        const Record &r = rec[i];
        if (r.q_start < 0 || r.q_len < 0 || r.k_start < 0 || r.k_len < 0 || r.k_len > kMaxRows ||
            r.q_len > kMaxRows / group)
            return -CT_EINVAL_SHAPE;
        tiles += cdiv(r.q_len * group, kTile) + cdiv(r.k_len, kTile);
    }
    if (tiles > 0x7fffffff / (4 * kTile * kv_heads)) return -CT_EINVAL_SHAPE;
    try {
        Plan made;
        make_plan(pass, rec, n_records, kv_heads, group, padded_dim(head_dim), causal != 0, dtype, made);
        counts[0] = (int64_t)made.pieces.size();
        counts[1] = (int64_t)made.joins.size();
        counts[2] = made.slots;
        counts[3] = (int64_t)made.groups.size();
        if (!counts_ok(counts, kv_heads)) return -CT_EINVAL_SHAPE;
        if (!entries) return 0;
        if (capacity < counts[0] + counts[1] + counts[3]) return -CT_EINVAL_WORKSPACE;
        Item *dst = std::copy(made.pieces.begin(), made.pieces.end(), reinterpret_cast<Item *>(entries));
        dst = std::copy(made.joins.begin(), made.joins.end(), dst);
        std::copy(made.groups.begin(), made.groups.end(), reinterpret_cast<Group *>(dst));
    } catch (...) {
        return (int)hipErrorOutOfMemory;
    }
    return 0;
}

extern "C" int64_t ct_attention_workspace(int32_t pass, int64_t slots, int32_t kv_heads, int32_t head_dim) {
    if (slots <= 0 || kv_heads <= 0 || head_dim <= 0 || head_dim > 128) return 0;
    return slots * kv_heads * parts_per_item(pass, padded_dim(head_dim)) * (int64_t)sizeof(float);
}

extern "C" int ct_attention_forward(const ct_attention *c, const int32_t *plan, const int64_t *counts, void *out,
                                    float *stats, void *workspace, int64_t workspace_bytes, hipStream_t stream) {
    AttnParams a;
    if (const int status = fill_params(c, a)) return status;
    if (!counts) return -CT_EINVAL_POINTER;
    if (!counts_ok(counts, c->kv_heads)) return -CT_EINVAL_SHAPE;
    const int64_t joins = counts[1], slots = counts[2], groups = counts[3];
    if (groups == 0) return 0;
    if (!plan || !out || (uintptr_t)plan % 16 || (uintptr_t)out % 16) return -CT_EINVAL_POINTER;
    if ((uintptr_t)stats % 8) return -CT_EINVAL_POINTER;
    if (slots && (!workspace || (uintptr_t)workspace % 16 ||
                  workspace_bytes < ct_attention_workspace(CT_ATTENTION_FORWARD, slots, c->kv_heads, c->head_dim)))
        return -CT_EINVAL_WORKSPACE;
    const int dp = padded_dim(c->head_dim);
    set_plan(a, plan, counts);
    a.dst0 = (char *)out;
    a.stats = (float2 *)stats;
    a.part0 = (float *)workspace;
    a.part1 = a.part0 + slots * c->kv_heads * kRowTile * dp;
    return by_type(c->dtype, dp, [&](auto type, auto dim) {
        typedef decltype(type) T;
        constexpr int DP = decltype(dim)::value;
        attention_forward<T, DP>
            <<<dim3((unsigned)(groups * c->kv_heads)), dim3(64 * kRowWaves), 0, stream>>>(a);
        if (const int status = status_of_last_launch()) return status;
        if (!joins) return 0;
        attention_join<T, DP><<<dim3((unsigned)(joins * c->kv_heads)), dim3(kThreads), 0, stream>>>(
            a, a.items + counts[0], kRowTile);
        return status_of_last_launch();
    });
}

extern "C" int ct_attention_backward(const ct_attention *c, const int32_t *row_plan, const int64_t *row_counts,
                                     const int32_t *key_plan, const int64_t *key_counts, const void *out,
                                     const float *stats, const void *dout, int64_t dout_token, int64_t dout_head,
                                     float *terms, void *dq, void *dk, void *dv, void *workspace,
                                     int64_t workspace_bytes, hipStream_t stream) {
    AttnParams a;
    if (const int status = fill_params(c, a)) return status;
    if (!row_counts || !key_counts) return -CT_EINVAL_POINTER;
    if (!counts_ok(row_counts, c->kv_heads) || !counts_ok(key_counts, c->kv_heads)) return -CT_EINVAL_SHAPE;
    const int64_t rows = row_counts[3], keys = key_counts[3], row_slots = row_counts[2], key_slots = key_counts[2];
    const int64_t size = c->dtype == CT_BF16 ? 2 : 4;
    if (rows) {
        if (!row_plan || !out || !stats || !dout || !terms || !dq ||
            ((uintptr_t)row_plan | (uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)terms) % 16 ||
            (uintptr_t)stats % 8)
            return -CT_EINVAL_POINTER;
        if (dout_token < 0 || dout_head < 0 || dout_token * size % 16 || dout_head * size % 16 ||
            dout_token > (int64_t)1 << 40 || dout_head > (int64_t)1 << 40)
            return -CT_EINVAL_SHAPE;
        if (!row_span_ok(dout_token * size, dout_head * size, a.group)) return -CT_EINVAL_SHAPE;
    }
    if (keys && (!key_plan || !dk || !dv || ((uintptr_t)key_plan | (uintptr_t)dk | (uintptr_t)dv) % 16))
        return -CT_EINVAL_POINTER;
    // the two passes use the workspace one after the other
    const int64_t needed = std::max(ct_attention_workspace(CT_ATTENTION_ROWS, row_slots, c->kv_heads, c->head_dim),
                                    ct_attention_workspace(CT_ATTENTION_KEYS, key_slots, c->kv_heads, c->head_dim));
    if (needed && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < needed)) return -CT_EINVAL_WORKSPACE;
    const int dp = padded_dim(c->head_dim);
    a.out = (const char *)out;
    a.dout = (const char *)dout;
    a.do_token = dout_token * size;
    a.do_head = dout_head * size;
    a.stats = (float2 *)const_cast<float *>(stats);
    a.terms = (float4 *)terms;
    return by_type(c->dtype, dp, [&](auto type, auto dim) {
        typedef decltype(type) T;
        constexpr int DP = decltype(dim)::value;
        AttnParams r = a;
        r.part0 = (float *)workspace;
        if (rows) {   // dq first: it leaves the rows' terms for the other kernel
            set_plan(r, row_plan, row_counts);
            r.dst0 = (char *)dq;
            r.d_token = a.o_token;
            attention_dq<T, DP>
                <<<dim3((unsigned)(rows * c->kv_heads)), dim3(64 * kRowWaves), 0, stream>>>(r);
            if (const int status = status_of_last_launch()) return status;
            if (row_counts[1]) {
                attention_dq_join<T, DP><<<dim3((unsigned)(row_counts[1] * c->kv_heads)), dim3(kThreads), 0, stream>>>(
                    r, r.items + row_counts[0], kRowTile);
                if (const int status = status_of_last_launch()) return status;
            }
        }
        if (!keys) return 0;
        set_plan(r, key_plan, key_counts);
        r.dst0 = (char *)dk;
        r.dst1 = (char *)dv;
        r.d_token = c->kv_heads * a.o_head;
        r.part1 = r.part0 + key_slots * c->kv_heads * kTile * DP;
        attention_dkv<T, DP><<<dim3((unsigned)(keys * c->kv_heads)), dim3(64 * kKeyWaves), 0, stream>>>(r);
        if (const int status = status_of_last_launch()) return status;
        if (!key_counts[1]) return 0;
        attention_dkv_join<T, DP><<<dim3((unsigned)(key_counts[1] * c->kv_heads)), dim3(kThreads), 0, stream>>>(
            r, r.items + key_counts[0]);
        return status_of_last_launch();
    });
}
