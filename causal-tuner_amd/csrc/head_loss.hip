// The head's loss over a large vocabulary, walked in pieces, gfx950: cross-entropy to one label,
// or to a teacher's top entries, of softmax(h W^T / T) without the logits ever being held.
//
// With l_iv = h_i . w_v / T, Z_i = sum_v exp(l_iv), a row's targets (v_k, q_k), k < K, distinct and
// sorted, mass Q = sum_k q_k and entropy term H = sum_k q_k log q_k:
//
//   loss  = sum_i c_i (H_i + sum_k q_ik (log Z_i - l_iv_k))
//   dh_i  = c_i / T (Q_i / Z_i sum_v exp(l_iv) w_v - sum_k q_ik w_v_k)
//   dW_v  = sum_i c_i / T (Q_i exp(l_iv) / Z_i - q_iv) h_i
//
// A hard label is K = 1, q = 1, H = 0. The hidden gradient is attention with the head as keys and
// values, so the forward makes it in the same sweep over the vocabulary, piece by piece: one
// product writes E = 2^(l log2 e - c), in one to three bf16 terms, beside the float32 sums of a running
// softmax; the next adds E W_piece to a float32 accumulator per row; Z divides at the end. The
// targets' own terms are left out of E and of the sums, and their coefficients Q p_k - q_k formed in
// double from their logits and the others' sum: for a label of probability near one, 1 - p is not the
// difference of two roundings. The backward adds them in float32. The head's gradient needs the
// finished Z: the backward forms the logits of a piece again, E becomes the derivative itself, and
// a second product multiplies it with the hidden rows.
//
// bf16. Both products run on v_mfma_f32_16x16x32_bf16 with one operand, the left one of every
// product, stored in the order in which the lanes take it ("packed": 1 KB per 16 rows x 32
// reduction indices, lane l's 16 bytes at 16 l), so that it goes from global memory to registers
// with whole-line loads and never through LDS; only the other operand is staged there. The logits
// kernel writes E packed for the product that follows straight from its accumulators: a lane holds
// 4 + 4 values of one row, which become one 16-byte unit. That fixes the order of the reduction
// indices inside a block of 32 (unit q holds indices 4 q .. + 3 and 16 + 4 q .. + 3), and the
// product that follows reads its LDS tile in that order.
//
// float32. Operands are split into three bf16 terms, which hold them exactly, and take the same
// kernels (Core, TRI).
//
// Bound by the matrix units from some 300 rows on: 4 rows vocab width operations with the hidden
// gradient, 8 with the head's too (2 of them the logits again, the price of not holding them). In bf16,
// 49152 entries x 2048: 16384 rows with the hidden gradient 5.5 ms, 1.19 PFLOP/s (a library product of
// such sizes alone runs at 1.26 to 1.55); 4001 rows with both gradients 2.8 ms, 1.15 PFLOP/s (logits 706
// and 713, products 623 and 660 us). Of few rows by a read of the head for each product, from HBM and
// in part from the last-level cache: one row, 201 MB, logits 33 us, product 34.
//
// Every sum runs in a fixed order: repeated calls are bit-identical.

#include <math.h>

#include <type_traits>

#include "gemm_common.hpp"
#include "term_steps.hpp"

namespace ct {
namespace {

constexpr int kStep = 64;              // reduction indices per step of a product
constexpr int kUnit = 128;             // vocabulary entries per (row, unit) pair of statistics
constexpr int kMaxEntries = 1024;
// bf16: up to so many rows, where reading the head bounds, the exponentials (twice as many: the
// derivative) are kept in two bf16 terms: one rounding, by up to 2^-8, of the one or two large values that a
// row has shows in the gradients of few rows. A head gradient of more rows is rounded twice, in the derivative and
// in the result (0.0024 of its norm for 0.0017); the derivative in two terms would cost 12% of the pass there (257
// rows x 32003 x 1000) to 21% (1000 rows and more).
constexpr int64_t kTwoTerms = 128;
constexpr int64_t kMaxPitch = 1 << 20;   // a tile's offsets stay below 2^31
// A launch holds fewer than 2^32 threads: 256 per row, one per eight values of the padded rows.
constexpr int64_t kMaxWidth = 65536, kMaxVocab = (int64_t{1} << 31) - 1024, kMaxRows = (int64_t{1} << 24) - 256;
constexpr int64_t kMaxValues = (int64_t{1} << 35) - 256;
// Rows of a head gradient: transposed, they are the columns of a tile's 256 rows of bf16, up(rows, kStep) apart,
// whose bytes a descriptor's 2^31 - 1 have to hold.
constexpr int64_t kMaxHeadRows = (0x7fffffff / (256 * 2)) / kStep * kStep;
// Values of one piece, in bytes, whatever the batch and the vocabulary. Larger pieces read and write the
// float32 sums less often (16384 tokens, of 49152 entries: 128 MB 6.25 ms, 256 MB 5.75, 512 MB 5.54, 1 GB
// 5.47), smaller ones stay in the 256 MB last-level cache, which pays for less than that.
constexpr int64_t kPieceBytes = int64_t{512} << 20;
constexpr float kNone = -3e38f;        // the shift of a row or unit without a finite logit
constexpr int kNoEntry = 0x7fffffff;

__host__ __device__ constexpr int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// ------------------------------------------------------------------------- plan of a call
struct Plan {
    int64_t rows, width, vocab, entries;
    int dtype, bp, bl;      // a workgroup's packed rows and vocabulary entries (or columns)
    int64_t rows_pad, width_pad, units;
    int64_t piece;          // vocabulary entries per piece of the sweep
    int splits;             // of the hidden gradient's reduction
    bool turned;            // the second products read their staged operand transposed
    bool tri;               // float32 in three bf16 terms
    int terms[3];           // bf16 terms of a piece's values, by sweep
    int chunks;             // of the logits' reduction; more than one: logits in memory, exponentials by row
};

// Workgroups' worth of work in whole rounds: how many splits of a reduction of `steps` leave the
// fewest compute units idle, each further split paying for another pass over the sums.
int splits_for(int64_t tiles, int64_t slots, int64_t steps) {
    int best = 1;
    double most = 0;
    for (int s = 1; s <= 64 && s <= (steps + 3) / 4; ++s) {
        const double work = (double)tiles * s, rounds = (double)((int64_t)(work + slots - 1) / slots);
        const double gain = work / (rounds * slots) - 0.02 * (s - 1) * (tiles >= 32 ? 1 : 0.1);
        if (gain > most + 1e-9) {
            most = gain;
            best = s;
        }
    }
    return best;
}

// Of `all` columns of tiles, how many make a piece: at most `most`, such that the rounds of
// workgroups over all pieces are fewest, each further piece paying for a pass over the sums. (2665
// rows and 192 columns of 11 tiles each: pieces of 186 and 6 columns run 9 rounds, two of 96 each 10.)
int64_t piece_for(int64_t all, int64_t most, int64_t rows, int64_t slots) {
    if (all <= most) return all;
    int64_t best = most;
    double least = 1e30;
    for (int64_t n = most; n > most / 2; --n) {
        const int64_t whole = all / n, rest = all % n;
        const double cost = (double)(whole * cdiv(n * rows, slots) + cdiv(rest * rows, slots)) + 0.5 * (whole + (rest > 0));
        if (cost < least - 1e-9) {
            least = cost;
            best = n;
        }
    }
    return best;
}

// A small vocabulary's logits are a few tiles, each a chain of the width's steps. Where they leave more
// than half of the compute units idle and the chain is worth cutting, it is cut: the logits, at most
// 128 tiles of them, go through memory. (18 rows x 328 entries x 3496, float32: 1.15 ms in one chain.)
int chunks_for(int64_t tiles, int64_t steps) {
    if (tiles > 128 || steps < 8) return 1;
    const int64_t idle = cdiv(256, tiles), most = steps / 4;
    return (int)(idle < most ? idle : most);
}

Plan plan_of(int64_t rows, int64_t width, int64_t vocab, int64_t entries, int dtype) {
    Plan p{};
    p.rows = rows;
    p.width = width;
    p.vocab = vocab;
    p.entries = entries;
    p.dtype = dtype;
    p.tri = dtype == CT_F32;
    // float32: the narrow tile, which splits the head on the way to LDS, up to where the wide ones' reuse
    // pays for terms in memory and transposes (with both gradients, narrow and wide: 500 rows x 4000 x 1000 183
    // and 386 us, 4000 x 2000 x 1000 540 and 1127, 500 x 32001 x 1022 1045 and 1070, 1000 x 16000 x 1000 980 and
    // 894, 2000 x 16000 x 1024 1825 and 1590).
    const bool narrow = rows <= 64 || (p.tri && (rows <= 512 || cdiv(rows, 64) * cdiv(vocab, 128) <= 1024));
    p.bp = narrow ? 64 : rows <= 128 ? 128 : 256;
    p.bl = p.bp == 64 ? 128 : 256;
    p.rows_pad = up(rows, p.bp);
    p.width_pad = up(width, kStep);
    p.units = cdiv(vocab, kUnit);
    p.terms[0] = 1;
    p.terms[1] = p.tri ? 3 : rows <= kTwoTerms ? 2 : 1;
    p.terms[2] = p.tri ? 3 : rows <= 2 * kTwoTerms ? 2 : 1;
    const int64_t element = 2 * p.terms[2];
    int64_t most = kPieceBytes / (p.rows_pad * element) / 256 * 256;
    if (most < 1024) most = 1024;
    p.piece = piece_for(cdiv(vocab, 256), most / 256, p.rows_pad / p.bp * (p.bp == 64 ? 2 : 1), p.bp == 64 ? 512 : 256) * 256;
    p.turned = p.tri ? p.bp > 64 : p.bp == 256;
    const int64_t tiles = p.rows_pad / p.bp * cdiv(width, p.bl);
    p.splits = splits_for(tiles, p.bp == 64 && !p.tri ? 512 : 256, p.piece / kStep);
    p.chunks = chunks_for(p.rows_pad / p.bp * cdiv(vocab, p.bl), p.width_pad / kStep);
    return p;
}

// Entries per piece of a sweep. Statistics alone: bounded by the pairs per row and unit.
int64_t sweep_piece(const Plan &p, int sweep) {
    if (sweep || p.tri) return p.piece;
    const int64_t all = up(p.vocab, 2 * kUnit), most = kPieceBytes / (p.rows_pad * 8) / 2 * 2 * kUnit;
    return all < most ? all : most;
}

// What a call keeps for its backward, and its scratch: regions of one buffer each.
struct Regions {
    int64_t at = 0;
    int64_t take(int64_t bytes) {
        const int64_t start = at;
        at += up(bytes, 256);
        return start;
    }
};
struct Kept {
    int64_t index, q, chosen, first, shift, total, weight, mass, entropy, sums, slots, place, bytes;
};
// Slots of the table that counts how often a row is given: at most half of them are taken.
int64_t slots_for(int64_t rows) {
    int64_t n = 2;
    while (n < 2 * rows) n *= 2;
    return n;
}
Kept kept_of(const Plan &p, bool hidden_grad) {
    Regions r;
    Kept k{};
    k.index = r.take(p.rows * p.entries * 4);
    k.q = r.take(p.rows * p.entries * 4);
    k.chosen = r.take(p.rows * p.entries * 4);       // the targets' logits, later their coefficients
    k.first = r.take(p.rows_pad * (p.units + 1) * 2);
    k.shift = r.take(p.rows_pad * 4);                // c
    k.total = r.take(p.rows_pad * 4);                // Z 2^-c
    k.weight = r.take(p.rows_pad * 4);
    k.mass = r.take(p.rows_pad * 4);
    k.entropy = r.take(p.rows_pad * 4);
    k.sums = r.take(hidden_grad ? (int64_t)p.splits * p.rows * p.width * 4 : 0);
    k.slots = r.take(hidden_grad ? slots_for(p.rows) * 8 : 0);   // a row of the loss each, then how often it is given
    k.place = r.take(hidden_grad ? p.rows * 4 : 0);              // a row's slot
    k.bytes = r.at;
    return k;
}
struct Scratch {
    int64_t packed, plain, piece, turned, split, logits, stats, factor, inverse, near, losses, bytes;
};
// sweep 0: statistics alone, 1: with the hidden gradient's sums, 2: the head's gradient.
Scratch scratch_of(const Plan &p, int sweep) {
    Regions r;
    Scratch s{};
    const int64_t terms = p.tri ? 6 : 2, pitch = up(p.width, 8), steps = up(p.rows, kStep);
    const int64_t piece = sweep_piece(p, sweep);
    s.packed = r.take(p.rows_pad * p.width_pad * terms);
    s.plain = r.take(sweep == 2 ? p.rows * p.width * (p.tri ? 4 : 2) : 0);
    s.piece = r.take(sweep ? p.rows_pad * p.piece * 2 * p.terms[sweep] : 0);
    s.turned = r.take(sweep && p.turned ? p.width * terms * (sweep == 1 ? p.piece : steps) : 0);
    s.split = r.take(p.tri && p.turned ? p.piece * pitch * terms : 0);
    s.logits = r.take(p.chunks > 1 ? p.chunks * p.rows * p.vocab * 4 : 0);
    s.stats = r.take(sweep == 2 || p.chunks > 1 ? 0 : piece / kUnit * p.rows_pad * 8);
    s.factor = r.take(p.rows_pad * 4);
    s.inverse = r.take(p.rows_pad * 4);
    s.near = r.take(p.rows_pad * 4);
    s.losses = r.take(p.rows * 8);
    s.bytes = r.at;
    return s;
}

// ------------------------------------------------------------------------- targets
struct Targets {
    const int64_t *rows;       // which rows of the tables, or null
    int64_t tokens;            // rows of the tables
    const int64_t *indices;    // [*, entries], row pitch ld
    const float *values;       // the teacher's logits, or null: hard labels
    const float *normalizer;   // the teacher's log normalizer per row, or null
    const float *weights;
    int64_t ld_indices, ld_values;
};

// How often each row of the tables is given: a row of the loss finds the slot of its table row, whichever of the
// equal ones claims it, and counts there. `slots` null: rows are not numbered.
struct Repeats {
    int *slots, *place;
    int64_t size;   // a power of two; the counts follow the slots
    // Thread u of a launch with at least `size` threads; before any call of `count`.
    __device__ __forceinline__ void clear(int64_t u) const {
        if (!slots || u >= size) return;
        slots[u] = -1;
        slots[size + u] = 0;
    }
    __device__ __forceinline__ void count(const int64_t *rows, int64_t row) const {
        int64_t at = (int64_t)((uint64_t)rows[row] * 0x9e3779b97f4a7c15u >> 32) & (size - 1);
        for (;; at = (at + 1) & (size - 1)) {   // ends: there are more slots than rows
            const int held = atomicCAS(slots + at, -1, (int)row);
            if (held == -1 || rows[held] == rows[row]) break;
        }
        atomicAdd(slots + size + at, 1);
        place[row] = (int)at;
    }
};

// A float sum over the workgroup, in a fixed order.
template <int THREADS>
__device__ __forceinline__ float block_sum(float v, float *lds) {
    lds[threadIdx.x] = v;
    __syncthreads();
    for (int h = THREADS / 2; h > 0; h >>= 1) {
        if (threadIdx.x < h) lds[threadIdx.x] += lds[threadIdx.x + h];
        __syncthreads();
    }
    const float sum = lds[0];
    __syncthreads();
    return sum;
}
template <int THREADS>
__device__ __forceinline__ float block_max(float v, float *lds) {
    lds[threadIdx.x] = v;
    __syncthreads();
    for (int h = THREADS / 2; h > 0; h >>= 1) {
        if (threadIdx.x < h) lds[threadIdx.x] = fmaxf(lds[threadIdx.x], lds[threadIdx.x + h]);
        __syncthreads();
    }
    const float top = lds[0];
    __syncthreads();
    return top;
}

// One workgroup per row: q of its entries, sorted by index with equal indices joined, the entries
// outside the vocabulary dropped; `first` [row][unit] counts the entries before each unit. Rows of
// the padding get no entries and no weight.
template <int THREADS, int MOST>
__global__ __launch_bounds__(THREADS) void targets_kernel(Targets t, int64_t rows, int entries, int64_t vocab,
                                                          int64_t units, double inverse_t, int *__restrict__ index,
                                                          float *__restrict__ q_out, float *__restrict__ chosen,
                                                          uint16_t *__restrict__ first, float *__restrict__ weight,
                                                          float *__restrict__ mass, float *__restrict__ entropy,
                                                          float *__restrict__ shift, float *__restrict__ total,
                                                          const Repeats repeats) {
    __shared__ uint64_t key[MOST];
    __shared__ float value[MOST], lds[THREADS];
    __shared__ int sorted[MOST], kept;
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    if (tid == 0) {
        shift[row] = kNone;
        total[row] = 0.f;
    }
    const int64_t from = row < rows && t.rows ? t.rows[row] : row;
    if (row >= rows || from < 0 || from >= t.tokens) {
        if (row < rows)
            for (int e = tid; e < entries; e += THREADS) {
                index[row * entries + e] = kNoEntry;
                q_out[row * entries + e] = chosen[row * entries + e] = 0.f;
            }
        for (int64_t u = tid; u <= units; u += THREADS) first[row * (units + 1) + u] = 0;
        if (tid == 0) weight[row] = mass[row] = entropy[row] = 0.f;
        return;
    }
    if (repeats.slots && tid == 0) repeats.count(t.rows, row);
    if (!t.values) {  // one hard label
        const int64_t label = t.indices[from * t.ld_indices];
        const bool there = label >= 0 && label < vocab;
        for (int64_t u = tid; u <= units; u += THREADS)
            first[row * (units + 1) + u] = there && label < u * kUnit ? 1 : 0;
        if (tid == 0) {
            index[row] = there ? (int)label : kNoEntry;
            q_out[row] = there ? 1.f : 0.f;
            chosen[row] = 0.f;
            weight[row] = t.weights[from];
            mass[row] = 1.f;
            entropy[row] = 0.f;
        }
        return;
    }
    int size = 1;
    while (size < entries) size <<= 1;
    float top = -INFINITY;
    for (int e = tid; e < size; e += THREADS) {
        uint64_t k = ~uint64_t{0};
        if (e < entries) {
            const int64_t at = t.indices[from * t.ld_indices + e];
            if (at >= 0 && at < vocab) {
                k = (uint64_t)at << 32 | (uint32_t)e;
                const float v = (float)((double)t.values[from * t.ld_values + e] * inverse_t);
                value[e] = v;
                top = fmaxf(top, v);
            }
        }
        key[e] = k;
    }
    if (t.normalizer) {
        top = t.normalizer[from];
    } else {
        top = block_max<THREADS>(top, lds);
        if (top == -INFINITY) top = 0.f;   // no entry holds any mass
    }
    __syncthreads();
    float sum = 0.f;
    for (int e = tid; e < entries; e += THREADS)
        if (key[e] != ~uint64_t{0}) {
            value[e] = value[e] - top;
            sum += expf(value[e]);
        }
    sum = block_sum<THREADS>(sum, lds);
    const float norm = t.normalizer || sum == 0.f ? 0.f : logf(sum);
    for (int width = 2; width <= size; width <<= 1)   // bitonic, ascending
        for (int stride = width / 2; stride > 0; stride >>= 1) {
            __syncthreads();
            for (int e = tid; e < size; e += THREADS) {
                const int other = e ^ stride;
                if (other > e) {
                    const uint64_t a = key[e], b = key[other];
                    if ((a > b) == ((e & width) == 0)) {
                        key[e] = b;
                        key[other] = a;
                    }
                }
            }
        }
    __syncthreads();
    // The first of equal indices takes their sum; its place is the count of firsts before it.
    if (tid < 64) {
        int n = 0;
        for (int base = 0; base < size; base += 64) {
            const int e = base + tid;
            const bool is = e < size && key[e] != ~uint64_t{0} && (e == 0 || (key[e] >> 32) != (key[e - 1] >> 32));
            const uint64_t all = __builtin_amdgcn_ballot_w64(is);
            if (is) sorted[n + __builtin_popcountll(all & ((uint64_t{1} << tid) - 1))] = e;
            n += __builtin_popcountll(all);
        }
        if (tid == 0) kept = n;
    }
    __syncthreads();
    float held = 0.f, ent = 0.f;
    for (int n = tid; n < entries; n += THREADS) {
        const int64_t to = row * entries + n;
        chosen[to] = 0.f;
        if (n >= kept) {
            index[to] = kNoEntry;
            q_out[to] = 0.f;
            continue;
        }
        const int e = sorted[n], at = (int)(key[e] >> 32);
        const int next = n + 1 < kept ? sorted[n + 1] : size;
        float log_q = value[(uint32_t)key[e]] - norm, q = expf(log_q);
        bool joined = false;
        for (int m = e + 1; m < next && (int)(key[m] >> 32) == at && key[m] != ~uint64_t{0}; ++m) {
            q += expf(value[(uint32_t)key[m]] - norm);
            joined = true;
        }
        if (joined) log_q = logf(q);
        index[to] = at;
        q_out[to] = q;
        held += q;
        if (q != 0.f) ent += q * log_q;
    }
    held = block_sum<THREADS>(held, lds);
    ent = block_sum<THREADS>(ent, lds);
    if (tid == 0) {
        weight[row] = t.weights[from];
        mass[row] = held;
        entropy[row] = ent;
    }
    for (int64_t u = tid; u <= units; u += THREADS) {
        int lo = 0, hi = kept;   // entries with an index below u * kUnit
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if ((int64_t)(key[sorted[mid]] >> 32) < u * kUnit) lo = mid + 1;
            else hi = mid;
        }
        first[row * (units + 1) + u] = (uint16_t)lo;
    }
}

// ------------------------------------------------------------------------- packing
// The row of `hidden` that row i of the loss is, or -1.
struct Source {
    const void *x;
    const int64_t *rows;
    int64_t ld, count, tokens, width;   // width: columns of x, zeros past them
    __device__ __forceinline__ int64_t row(int64_t i) const {
        if (i >= count) return -1;
        const int64_t r = rows ? rows[i] : i;
        return r >= 0 && r < tokens ? r : -1;
    }
};

// Eight float32 values as sums of bf16 terms, 8 bits of the significand each, term by term as 16-byte
// units: three terms hold values of 2^-100 and more exactly.
template <int TERMS>
__device__ __forceinline__ void split_unit(const float (&v)[8], uint4 (&out)[TERMS]) {
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = v[i];
#pragma unroll
    for (int s = 0; s < TERMS; ++s) {
        out[s] = make_uint4(pack_bf16x2(rest[0], rest[1]), pack_bf16x2(rest[2], rest[3]), pack_bf16x2(rest[4], rest[5]),
                            pack_bf16x2(rest[6], rest[7]));
        if (s + 1 == TERMS) break;
        const uint32_t w[4] = {out[s].x, out[s].y, out[s].z, out[s].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] -= bf16_to_f32((uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
    }
}

// pack_rows below for float32 rows: three packed operands, `units` apart.
__global__ __launch_bounds__(256) void pack_split(Source src, int64_t blocks, uint4 *__restrict__ out, int64_t units,
                                                  const Repeats repeats) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= units) return;
    repeats.clear(u);
    const int lane = (int)(u & 63);
    const int64_t block = u >> 6, kb = block % blocks, row = src.row(block / blocks * 16 + (lane & 15));
    const int64_t k = kb * 32 + (lane >> 4) * 8;
    const float *x = static_cast<const float *>(src.x) + row * src.ld;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = row >= 0 && k + i < src.width ? x[k + i] : 0.f;
    uint4 t[3];
    split_unit<3>(v, t);
#pragma unroll
    for (int s = 0; s < 3; ++s) out[u + s * units] = t[s];
}

// float32 rows [rows][cols] as three bf16 arrays of `pitch` columns, `apart` units between them.
template <bool PAIRS>
__global__ __launch_bounds__(256) void split_rows(const float *__restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                  uint4 *__restrict__ out, int64_t pitch, int64_t apart) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x, per = pitch / 8, row = u / per, c = u % per * 8;
    if (row >= rows) return;
    float v[8];
    if (PAIRS && c + 8 <= cols) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 f = *reinterpret_cast<const float2 *>(x + row * ld + c + i);
            v[i] = f.x, v[i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? x[row * ld + c + i] : 0.f;
    }
    uint4 t[3];
    split_unit<3>(v, t);
#pragma unroll
    for (int s = 0; s < 3; ++s) out[u + s * apart] = t[s];
}

// Hidden rows in the order of a product's packed operand, zeros past the rows and the width. On the way the
// slots of `repeats` are cleared: eight units or more a row, four slots at most.
template <bool VEC>
__global__ __launch_bounds__(256) void pack_rows(Source src, int64_t blocks, uint4 *__restrict__ out, int64_t units,
                                                 const Repeats repeats) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= units) return;
    repeats.clear(u);
    const int lane = (int)(u & 63);
    const int64_t block = u >> 6, kb = block % blocks, row = src.row(block / blocks * 16 + (lane & 15));
    const int64_t k = kb * 32 + (lane >> 4) * 8;
    const uint16_t *x = static_cast<const uint16_t *>(src.x) + row * src.ld;
    uint4 v = zero4();
    if (row >= 0) {
        if constexpr (VEC) {
            if (k < src.width) v = *reinterpret_cast<const uint4 *>(x + k);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < src.width) w[i / 2] |= (uint32_t)x[k + i] << (16 * (i & 1));
            v = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    out[u] = v;
}

// The same rows one after the other, `pitch` columns each.
template <class T>
__global__ __launch_bounds__(256) void gather_rows(Source src, T *__restrict__ out, int64_t pitch) {
    const int64_t row = src.row(blockIdx.x);
    const T *x = static_cast<const T *>(src.x) + row * src.ld;
    for (int64_t c = threadIdx.x; c < pitch; c += 256)
        out[blockIdx.x * pitch + c] = row >= 0 && c < src.width ? x[c] : T(0);
}

// out [cols][pitch] = x [rows][cols] transposed, the indices inside each block of 32 rows in the
// order of the second product (unit q: 4 q .. + 3, 16 + 4 q .. + 3), zeros past the rows. A workgroup
// takes 64 x 64. Bound by the copy (49152 x 2048 bf16: 74 us, 5.4 TB/s), which of more than 128 rows costs less
// than the product's transposing reads from LDS. float32: three bf16 arrays, `apart` units between them.
template <class T>
__global__ __launch_bounds__(256) void transpose_rows(const T *__restrict__ x, int64_t ld, int64_t rows, int64_t cols,
                                                      uint4 *__restrict__ out, int64_t pitch, int64_t apart) {
    constexpr int PER = 16 / sizeof(T), UNITS = 64 * 64 / PER;
    __shared__ T tile[64][64 + PER];
    const int64_t r0 = (int64_t)blockIdx.x * 64, c0 = (int64_t)blockIdx.y * 64;
#pragma unroll
    for (int i = 0; i < UNITS / 256; ++i) {
        const int u = threadIdx.x + i * 256, r = u / (64 / PER), c = u % (64 / PER) * PER;
        if constexpr (sizeof(T) == 2) {   // rows of whole units
            uint4 v = zero4();
            if (r0 + r < rows && c0 + c < cols) v = *reinterpret_cast<const uint4 *>(x + (r0 + r) * ld + c0 + c);
            *reinterpret_cast<uint4 *>(&tile[r][c]) = v;
        } else {
#pragma unroll
            for (int e = 0; e < PER; ++e)
                tile[r][c + e] = r0 + r < rows && c0 + c + e < cols ? x[(r0 + r) * ld + c0 + c + e] : 0.f;
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int u = threadIdx.x + i * 256, c = u >> 3, unit = u & 7, from = (unit >> 2) * 32 + (unit & 3) * 4;
        if (c0 + c >= cols) continue;
        uint4 *to = out + ((c0 + c) * pitch + r0) / 8 + unit;
        if constexpr (sizeof(T) == 2) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = from + (j >> 1) * 16 + (j & 1) * 2;
                w[j] = (uint32_t)tile[r][c] | (uint32_t)tile[r + 1][c] << 16;
            }
            *to = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = tile[from + (j >> 2) * 16 + (j & 3)][c];
            uint4 t[3];
            split_unit<3>(v, t);
#pragma unroll
            for (int s = 0; s < 3; ++s) to[s * apart] = t[s];
        }
    }
}

// ------------------------------------------------------------------------- the product's core
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// What workgroup `id` of `total` comes to when each of the 8 XCDs walks a contiguous range.
__device__ __forceinline__ int64_t by_xcd(int64_t id, int64_t total) {
    const int64_t share = total / 8, more = total % 8, x = id & 7, i = id >> 3;
    return x < more ? x * (share + 1) + i : more * (share + 1) + (x - more) * share + i;
}
// Tile t of np x nl, in groups of four packed tiles that share the other operand's tile in an L2.
__device__ __forceinline__ void tile_at(int64_t t, int64_t np, int64_t nl, int64_t &tp, int64_t &tl) {
    const int64_t size = 4 * nl, group = t / size, at = t - group * size;
    const int64_t count = np - group * 4 < 4 ? np - group * 4 : 4;
    tp = group * 4 + at % count;
    tl = at / count;
}

// acc[f][j] += fragment f of the staged operand x fragment j of the packed one, over the reduction.
// WP x WL waves, each of PF x LF fragments of 16. KT: the staged operand is stored with the reduction
// index as its row (as values in attention are), in LDS too, and its fragments come from transposing
// reads; else its rows are reduction-contiguous. SWAP: the staged operand is the MFMA's first, so a
// lane holds four of its consecutive rows for one packed row; otherwise four packed rows for one of
// the staged ones.
//
// A step of 64 indices runs column by column (a fragment of the staged operand against all packed
// ones), the order of everything in it fixed: a column's fragments are read three columns ahead, the
// first three of the next step's at the end of this one, which its third stage allows, and the packed
// fragments loaded two steps ahead; the loads and
// the stores of the tiles to come lie one by one between the columns. (In one run each, all waves queue
// behind them: 3% slower.) Eight waves side by side along the packed rows read no packed row twice;
// 4 x 2 waves, with half the LDS reads and twice the packed loads, are 6% slower, two workgroups of four
// waves per CU 9%.
//
// TERMS 2: the packed operand is the sum of two bf16 terms, both multiplied with each staged fragment.
// TERMS 3 (TRI): float32 operands as three bf16 terms each (split3). The reduction runs over six products of
// the terms, the small ones first; the three left out are below 2^-26 of the whole, and every
// product of two terms is exact in float32. Six bf16 products are faster than one float32 product
// on this card's matrix units (v_mfma_f32_16x16x4_f32, a sixteenth of the bf16 rate). The packed
// operand's terms, and on the wide tiles the staged one's, lie in memory one after the other (TRI, six
// passes over the reduction); the narrow tile, for few rows or tiles (plan_of), takes the staged one as
// float32, splits it on the way to LDS and makes the six products of a step together (FUSED: 3 rows x
// 60000 x 2000 0.78 ms, 1.70 with the terms in memory).
template <int WP, int WL, int PF, int LF, bool KT, bool SWAP, int TERMS = 1>
struct Core {
    static constexpr bool FUSED = TERMS == 3 && PF == 1 && LF == 8, TRI = TERMS == 3 && !FUSED;
    static constexpr int KS = TERMS == 2 ? 4 : FUSED ? 6 : 2;   // packed fragments of a step
    static constexpr int ES = FUSED ? 4 : 2, ST = FUSED ? 3 : 1;   // bytes of a staged value, terms in LDS
    static constexpr int BP = WP * PF * 16, BL = WL * LF * 16, THREADS = 64 * WP * WL;
    static constexpr int kPer = BL * 8 / THREADS;   // units (8 values) of a stage per thread
    static constexpr int kRaw = kPer * ES / 2;      // 16-byte loads of them
    static constexpr int kTerm = BL * 8, kStage = kTerm * ST;   // 16-byte units in LDS
    static constexpr int kRows = KT ? THREADS / (BL / 8) : THREADS / 8;   // rows between a thread's units
    static_assert(kRows % 16 == 0, "a thread's units differ by immediate offsets");

    const char *base;        // the staged operand at step 0 ...
    int64_t bytes, advance;  // ... the bytes from there to its end, and from one step to the next
    uint32_t off, pitch;     // of the thread's first unit, and between its units
    int k, limit;            // KC: the unit's first index of a step, and the depth
    const uint4 *a;          // the wave's packed rows at step 0
    int64_t a_row;           // units between two blocks of packed rows
    int steps, store_at, read_at;
    int one;                 // TRI: the steps of one product of terms
    TermDivisor part;        // TRI: the division by those
    int64_t b_apart, a_apart = 0;  // bytes, and units, between two terms

    // first: the staged operand at the tile's first row (KC) or column (KT); `extent` its rows from
    // there (KC) or columns (KT), `depth` the reduction's extent.
    __device__ __forceinline__ void init(const void *first, int64_t ld, int64_t extent, int64_t depth,
                                         const uint4 *packed, int64_t block, int64_t blocks, int wave) {
        const int tid = threadIdx.x, lane = tid & 63, wp = wave % WP, wl = wave / WP;
        base = static_cast<const char *>(first);
        limit = (int)depth;
        steps = (int)cdiv(depth, kStep);
        pitch = (uint32_t)(kRows * ld * ES);
        if constexpr (KT) {
            const int row = tid / (BL / 8), chunk = tid % (BL / 8), j = lane & 15, from = 4 * (lane >> 4) + (j >> 2);
            // bf16 rows are whole units
            bytes = ((depth - 1) * ld + (extent < BL ? FUSED ? extent : up(extent, 8) : BL)) * ES;
            advance = kStep * ld * ES;
            off = chunk * 8 < extent ? (uint32_t)((row * ld + chunk * 8) * ES) : kOOB;
            k = 0;
            store_at = row * (BL / 8) + ((chunk >> 1 ^ (row & 7)) << 1 | (chunk & 1));
            read_at = from * (BL * 2) + ((wl * LF ^ (from & 7)) << 5) + ((j & 3) << 3);
        } else {
            const int row = tid >> 3, chunk = tid & 7;
            // bf16 rows are whole units; rows past the extent lie behind the last
            bytes = (((extent < BL ? extent : BL) - 1) * ld + (FUSED ? depth : up(depth, 8))) * ES;
            advance = kStep * ES;
            off = (uint32_t)((row * ld + chunk * 8) * ES);
            k = chunk * 8;
            store_at = slot(row, chunk);
            read_at = slot(wl * LF * 16 + (lane & 15), lane >> 4);
        }
        a = packed + (block + wp * PF) * blocks * 64 + lane;
        a_row = blocks * 64;
    }
    __device__ __forceinline__ void terms(int64_t b_units, int64_t a_units) {
        a_apart = a_units;
        if constexpr (!TRI) return;
        one = steps;
        part = term_divisor(one);
        steps *= 6;
        b_apart = b_units * 16;
    }
    // The product of terms that step t belongs to, and the step in it. Of the packed operand the terms
    // 2 1 0 1 0 0, of the staged one 0 1 2 0 1 0.
    __device__ __forceinline__ int product(int t, int &at) const {
        const TermStep step = term_step(t, one, part);
        at = step.at;
        return step.product;
    }
    // The thread's unit C of step t, its fragment I, and the unit's place in a stage.
    template <int C>
    __device__ __forceinline__ void load_b(int t, uint4 (&r)[kRaw]) const {
        const char *from = base;
        int at = t;
        if constexpr (TRI) from += (0x124 >> 2 * product(t, at) & 3) * b_apart;
        // a descriptor per step: offsets stay within a step, whatever the operand's size
        const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(from + at * advance, t < steps ? bytes - at * advance : 0);
        const uint32_t to = (KT || at * kStep + k < limit ? off : kOOB) + C * pitch;
        if constexpr (FUSED) {
            r[2 * C] = buf_load16(rsrc, to);
            r[2 * C + 1] = buf_load16(rsrc, to + 16);
        } else {
            r[C] = buf_load16(rsrc, to);
        }
    }
    template <int I>
    __device__ __forceinline__ void load_a(int t, uint4 (&f)[KS][PF]) const {
        const uint4 *from = a;
        int at = t < steps ? t : steps - 1;
        if constexpr (TRI) from += (0x46 >> 2 * product(at, at) & 3) * a_apart;
        f[I % KS][I / KS] = from[(I % KS >> 1) * a_apart + (int64_t)at * 128 + I / KS * a_row + (I & 1) * 64];
    }
    template <int C>
    __device__ __forceinline__ void store_b(int t, uint4 *stage, const uint4 (&r)[kRaw]) const {
        const int to = store_at + C * kRows * (KT ? BL / 8 : 8);
        if constexpr (FUSED) {
            const uint32_t w[8] = {r[2 * C].x, r[2 * C].y, r[2 * C].z, r[2 * C].w,
                                   r[2 * C + 1].x, r[2 * C + 1].y, r[2 * C + 1].z, r[2 * C + 1].w};
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)   // a row's last unit reaches into the next row
                v[i] = KT || t * kStep + k + i < limit ? __builtin_bit_cast(float, w[i]) : 0.f;
            uint4 terms[3];
            split_unit<3>(v, terms);
#pragma unroll
            for (int s = 0; s < 3; ++s) stage[to + s * kTerm] = terms[s];
        } else {
            stage[to] = r[C];
        }
    }
    __device__ __forceinline__ void read(const uint4 *stages, int f, uint4 (&lf)[2 * ST]) const {
#pragma unroll
        for (int i = 0; i < 2 * ST; ++i) {
            const int ks = i & 1;
            const uint4 *stage = stages + (i >> 1) * kTerm;
            if constexpr (KT) {
                const __attribute__((address_space(3))) char *p =
                    (const __attribute__((address_space(3))) char *)stage + (read_at ^ (f & 7) << 5) + (f >> 3) * 256 + ks * 32 * (BL * 2);
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)p);
                const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(p + 16 * (BL * 2)));
                const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
                lf[i] = make_uint4(l2.x, l2.y, h2.x, h2.y);
            } else {
                lf[i] = stage[(read_at ^ ks << 2) + f * 128];
            }
        }
    }
    template <int F>
    __device__ __forceinline__ void columns(int t, const uint4 *cur, const uint4 *nxt, uint4 *wr, const uint4 (&af)[KS][PF],
                                            uint4 (&an)[KS][PF], uint4 (&b)[kRaw], uint4 (&lf)[4][2 * ST],
                                            f32x4 (&acc)[LF][PF]) const {
        if constexpr (F < LF) {
            read(F + 3 < LF ? cur : nxt, (F + 3) % LF, lf[(F + 3) % 4]);
            if constexpr (F % (LF / 8) == 0 && F / (LF / 8) < KS * PF) load_a<F / (LF / 8)>(t + 2, an);
            if constexpr (F % (LF / 4) == LF / 8 - 1) store_b<F / (LF / 4)>(t + 2, wr, b);
            if constexpr (F % (LF / 4) == LF / 4 - 1) load_b<F / (LF / 4)>(t + 3, b);
            // FUSED: of the packed operand the terms 2 1 0 1 0 0, of the staged one 0 1 2 0 1 0
#pragma unroll
            for (int m = 0; m < (FUSED ? 12 : KS); ++m) {
                const int x = FUSED ? (0x46 >> m / 2 * 2 & 3) * 2 + (m & 1) : m;
                const int y = FUSED ? (0x124 >> m / 2 * 2 & 3) * 2 + (m & 1) : m & 1;
#pragma unroll
                for (int j = 0; j < PF; ++j)
                    acc[F][j] = SWAP ? mfma16x16x32(lf[F % 4][y], af[x][j], acc[F][j])
                                     : mfma16x16x32(af[x][j], lf[F % 4][y], acc[F][j]);
            }
            __builtin_amdgcn_sched_barrier(0);
            columns<F + 1>(t, cur, nxt, wr, af, an, b, lf, acc);
        }
    }
    __device__ __forceinline__ void step(int t, uint4 *stages, int &at, const uint4 (&af)[KS][PF], uint4 (&an)[KS][PF],
                                         uint4 (&b)[kRaw], uint4 (&lf)[4][2 * ST], f32x4 (&acc)[LF][PF]) const {
        const int next = at == 2 * kStage ? 0 : at + kStage, after = next == 2 * kStage ? 0 : next + kStage;
        columns<0>(t, stages + at, stages + next, stages + after, af, an, b, lf, acc);
        static_assert(LF % 4 == 0, "the next step's first columns are in their places");
        at = next;
        __syncthreads();
    }
    template <int I>
    __device__ __forceinline__ void first(uint4 *stages, uint4 (&b)[kRaw], uint4 (&more)[kRaw], uint4 (&af)[KS][PF], uint4 (&ag)[KS][PF]) const {
        static_assert(kPer == 4 && KS * PF <= 8, "spread over the columns");
        if constexpr (I < 4) {
            load_b<I>(0, b);
            load_b<I>(1, more);
        } else if constexpr (I < 12) {
            if constexpr (I - 4 < KS * PF) { load_a<I - 4>(0, af); load_a<I - 4>(1, ag); }
        } else if constexpr (I < 16) {
            store_b<I - 12>(0, stages, b);
            store_b<I - 12>(1, stages + kStage, more);
            load_b<I - 12>(2, b);
        }
        if constexpr (I < 15) first<I + 1>(stages, b, more, af, ag);
    }
    __device__ __forceinline__ void run(uint4 *stages, f32x4 (&acc)[LF][PF]) const {
#pragma unroll
        for (int f = 0; f < LF; ++f)
#pragma unroll
            for (int j = 0; j < PF; ++j) acc[f][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (steps <= 0) return;
        uint4 b[kRaw], more[kRaw], a0[KS][PF], a1[KS][PF], a2[KS][PF], lf[4][2 * ST];
        first<0>(stages, b, more, a0, a1);
        __syncthreads();
        read(stages, 0, lf[0]);
        read(stages, 1, lf[1]);
        read(stages, 2, lf[2]);
        int t = 0, at = 0;
        for (; t + 2 < steps; t += 3) {
            step(t, stages, at, a0, a2, b, lf, acc);
            step(t + 1, stages, at, a1, a0, b, lf, acc);
            step(t + 2, stages, at, a2, a1, b, lf, acc);
        }
        if (t < steps) step(t, stages, at, a0, a2, b, lf, acc);
        if (t + 1 < steps) step(t + 1, stages, at, a1, a0, b, lf, acc);
    }
};

// ------------------------------------------------------------------------- logits of a piece
enum { STATS = 0, EXP = 1, GRAD = 2 };

struct LogitsParams {
    const void *head;          // from v0 on
    int64_t ld, width;
    int64_t head_apart, packed_apart, piece_apart;   // units between two terms
    const uint4 *packed;       // hidden rows
    int64_t blocks;            // of 32 along the width
    int64_t v0, v1;            // the piece's entries
    int64_t np, nl;            // tiles
    float scale;               // log2(e) / T
    uint4 *piece;              // EXP: E, GRAD: the derivative, packed
    int64_t piece_blocks;      // EXP: of 32 entries; GRAD: of 32 rows
    float2 *stats;             // [unit of the piece][row]
    int64_t rows_pad, rows;
    const int *index;
    const uint16_t *first;
    float *chosen;             // the targets' logits (written); GRAD: their coefficients (read)
    int entries;
    int64_t units;
    const float *shift, *factor, *inverse;   // GRAD: of row_factors
};

// The shift of a unit whose largest scaled logit is `top` (a whole number): one of ..., -128, -32,
// 64, ..., at most 80 below it and less than 16 above, so that units whose largest logits lie within
// 33 of zero share theirs and nothing is rescaled. E reaches 2^80, and holds what is down to 2^-110 of
// the unit's maximum.
__device__ __forceinline__ float shift_of(float top) {
    return fabsf(top) < 1e6f ? 96.f * ceilf((top - 48.f) * (1.f / 96.f)) - 32.f : top;
}

template <int TERMS>
__device__ __forceinline__ void store_unit(uint4 *to, int64_t apart, const float (&v)[8]) {
    uint4 t[TERMS];
    split_unit(v, t);
#pragma unroll
    for (int s = 0; s < TERMS; ++s) to[s * apart] = t[s];
}

// Which of a wave's rows x units of 128 vocabulary entries are targets, as bits in LDS [row][unit][4],
// a lane per row and unit.
template <int ROWS, int UNITS>
__device__ __forceinline__ void mark_targets(const LogitsParams &p, int64_t row0, int64_t unit0, uint32_t *bits, int lane) {
    static_assert(ROWS * UNITS <= 64, "a lane each");
    if (lane < ROWS * UNITS) {
        uint32_t w[4] = {0, 0, 0, 0};
        const int64_t row = row0 + lane / UNITS, unit = unit0 + lane % UNITS;
        if (row < p.rows && unit < p.units) {
            const uint16_t *at = p.first + row * (p.units + 1) + unit;
            for (int e = at[0]; e < at[1]; ++e) {
                const int v = p.index[row * p.entries + e] & (kUnit - 1);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (v >> 5 == i) w[i] |= 1u << (v & 31);
            }
        }
        *reinterpret_cast<uint4 *>(bits + lane * 4) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// The place among a row's sorted entries of the one at `bit` (0 .. 127) of unit `unit`.
__device__ __forceinline__ int64_t place_of(const LogitsParams &p, int64_t row, int64_t unit, const uint32_t *bits, int bit) {
    int n = p.first[row * (p.units + 1) + unit];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i <= bit >> 5) n += __builtin_popcount(i < bit >> 5 ? bits[i] : bits[i] & ((1u << (bit & 31)) - 1));
    return row * p.entries + n;
}

// A tile's logits from Core, and from the accumulators what MODE asks for, so that no logit reaches
// memory: the units' statistics (STATS), with E (EXP), or the derivative (GRAD), E and derivative in the
// order in which the product that follows takes them. The orientation follows from that order: a lane
// holds four entries of a row (EXP), or four rows of an entry (GRAD). 4001 rows x 49152 x 2048: 706 us,
// 1.14 PFLOP/s, of which a fifth to a quarter are the exponentials and the stores behind the product's last step, which
// workgroups that stay resident and overlap them did not hide (3% slower).
template <int WP, int WL, int PF, int LF, int MODE, int TERMS>
__global__ __launch_bounds__(64 * WP * WL) void logits_kernel(const LogitsParams p) {
    constexpr bool TRI = TERMS == 3;
    using C = Core<WP, WL, PF, LF, false, MODE != GRAD, TRI ? 3 : 1>;
    constexpr int UNITS = LF / 8;   // of a wave
    __shared__ uint4 stages[3 * C::kStage];
    __shared__ uint4 marks[WP * WL][PF * 16 * UNITS];
    int64_t tp, tl;
    tile_at(by_xcd(blockIdx.x, p.np * p.nl), p.np, p.nl, tp, tl);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % WP, wl = wave / WP, q = lane >> 4;
    const int64_t v0 = p.v0 + tl * C::BL, left = p.v1 - v0;
    const int64_t row0 = tp * C::BP + wp * PF * 16;
    uint32_t *wave_bits = reinterpret_cast<uint32_t *>(marks[wave]);
    mark_targets<PF * 16, UNITS>(p, row0, (v0 + wl * LF * 16) / kUnit, wave_bits, lane);
    C core;
    core.init(static_cast<const char *>(p.head) + (v0 - p.v0) * p.ld * C::ES, p.ld, left, p.width, p.packed, tp * (C::BP / 16), p.blocks, wave);
    if constexpr (TRI) core.terms(p.head_apart, p.packed_apart);
    f32x4 acc[LF][PF];
    core.run(stages, acc);

    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the lanes read each other's marks

#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        const int64_t u0 = v0 + (wl * UNITS + u) * kUnit, unit = u0 / kUnit;
        const int valid = (int)(p.v1 - u0 < kUnit ? (p.v1 > u0 ? p.v1 - u0 : 0) : kUnit);
        if constexpr (MODE == GRAD) {
            // lane: entry l % 16 of fragment f, rows 4 q + i of packed fragment j
#pragma unroll
            for (int j = 0; j < PF; ++j) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int local = j * 16 + 4 * q + i;
                    const int64_t row = row0 + local;
                    const float c = p.shift[row], factor = p.factor[row];
#pragma unroll
                    for (int f = 0; f < 8; ++f) {
                        const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[8 * u + f][j][i], p.scale, -c)) * factor;
                        acc[8 * u + f][j][i] = 16 * f + (lane & 15) < valid ? e : 0.f;
                    }
                    const uint32_t *bits = wave_bits + (local * UNITS + u) * 4;
                    const uint4 m = *reinterpret_cast<const uint4 *>(bits);
                    const uint32_t w[4] = {m.x, m.y, m.z, m.w};
                    if (__builtin_amdgcn_ballot_w64(((w[0] | w[1] | w[2] | w[3]) >> (lane & 15) & 0x00010001u) != 0)) {
                        const float inverse = p.inverse[row];   // 0 past the rows, which have no targets
#pragma unroll
                        for (int f = 0; f < 8; ++f) {
                            const int bit = 16 * f + (lane & 15);
                            if (w[f >> 1] >> (bit & 31) & 1)
                                acc[8 * u + f][j][i] = inverse * p.chosen[place_of(p, row, unit, bits, bit)];
                        }
                    }
                }
            }
#pragma unroll
            for (int f = 0; f < 8; ++f) {
                uint4 *to = p.piece + (((u0 - p.v0) / 16 + f) * p.piece_blocks + row0 / 32) * 64 + lane;
                if constexpr (PF == 1) {   // half a unit: the other half is the wave's that holds the next 16 rows
                    const f32x4 x = acc[8 * u + f][0];
                    uint4 t[TERMS];
                    split_unit({x[0], x[1], x[2], x[3]}, t);
#pragma unroll
                    for (int s = 0; s < TERMS; ++s)
                        reinterpret_cast<uint2 *>(to + s * p.piece_apart)[(row0 / 16) & 1] = make_uint2(t[s].x, t[s].y);
                } else {
#pragma unroll
                    for (int j = 0; j < PF; j += 2) {
                        const f32x4 x = acc[8 * u + f][j], y = acc[8 * u + f][j + 1];
                        store_unit<TERMS>(to + j / 2 * 64, p.piece_apart, {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]});
                    }
                }
            }
        } else {
            // lane: row l % 16 of packed fragment j, entries 4 q + i of fragment f
            if (valid < kUnit) {
#pragma unroll
                for (int f = 0; f < 8; ++f)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (16 * f + 4 * q + i >= valid)
#pragma unroll
                            for (int j = 0; j < PF; ++j) acc[8 * u + f][j][i] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < PF; ++j) {
                const int local = j * 16 + (lane & 15);
                const int64_t row = row0 + local;
                const uint32_t *bits = wave_bits + (local * UNITS + u) * 4;
                const uint4 m = *reinterpret_cast<const uint4 *>(bits);
                const uint32_t w[4] = {m.x, m.y, m.z, m.w};
                float top = acc[8 * u][j][0];
#pragma unroll
                for (int f = 0; f < 8; ++f)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = fmaxf(top, acc[8 * u + f][j][i]);
                top = fmaxf(top, __shfl_xor(top, 16, 64));
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                // exponents are taken relative to the unit's own maximum, where they are exact to
                // their own size, and brought to the shift by a power of two
                const float near = fmaxf(ceilf(top * p.scale), kNone), c = shift_of(near);
                const float by = near == c ? 1.f : ldexpf(1.f, (int)(near - c));
                float sum = 0.f;
#pragma unroll
                for (int g = 0; g < 4; ++g) {   // 32 entries: two fragments
                    float e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[8 * u + 2 * g + i / 4][j][i % 4], p.scale, -near));
                    const uint32_t mine = w[g] >> (4 * q) & 0x000f000fu;
                    if (mine) {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (mine >> (16 * (i / 4) + i % 4) & 1) {
                                p.chosen[place_of(p, row, unit, bits, 32 * g + 16 * (i / 4) + 4 * q + i % 4)] =
                                    acc[8 * u + 2 * g + i / 4][j][i % 4];
                                e[i] = 0.f;
                            }
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        sum += e[i];
                        e[i] *= by;
                    }
                    if constexpr (MODE == EXP)
                        store_unit<TERMS>(p.piece + ((row0 / 16 + j) * p.piece_blocks + (u0 - p.v0) / 32 + g) * 64 + lane,
                                        p.piece_apart, e);
                }
                sum += __shfl_xor(sum, 16, 64);
                sum += __shfl_xor(sum, 32, 64);
                if (q == 0) p.stats[(u0 - p.v0) / kUnit * p.rows_pad + row] = make_float2(c, sum * by);
            }
        }
    }
}

// The units' statistics of a piece joined to the rows': 16 rows x 64 groups of units a workgroup, in
// order (one row, 384 units: 6 us).
// A row's shift becomes the largest of its own and the units'; E of a unit with another shift is
// brought to it, and `factor` is what the sums of the pieces before are brought to it with.
__global__ __launch_bounds__(1024) void join_kernel(const float2 *__restrict__ stats, int units, int64_t rows_pad,
                                                   float *__restrict__ shift, float *__restrict__ total,
                                                   float *__restrict__ factor, uint4 *piece, int64_t piece_blocks,
                                                    int terms, int64_t apart) {
    __shared__ float part[64][17];
    const int r = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int64_t row = (int64_t)blockIdx.x * 16 + r;
    const float2 *at = stats + row;
    float c = kNone;
    for (int u = g; u < units; u += 64) c = fmaxf(c, at[u * rows_pad].x);
    part[g][r] = c;
    __syncthreads();
    const float before = shift[row], held = total[row];
    c = before;
#pragma unroll
    for (int i = 0; i < 64; ++i) c = fmaxf(c, part[i][r]);
    __syncthreads();
    float sum = 0.f;
    for (int u = g; u < units; u += 64) {
        const float2 s = at[u * rows_pad];
        if (s.x == c) {
            sum += s.y;
            continue;
        }
        const float by = __builtin_amdgcn_exp2f(s.x - c);
        sum += s.y * by;
        if (!piece) continue;
        for (int i = 0; i < kUnit / 8 * terms; ++i) {   // the row's 16 units of 16 bytes, term by term
            uint4 *e = piece + i / 16 * apart + (row / 16 * piece_blocks + u * (kUnit / 32) + i % 16 / 4) * 64 + i % 4 * 16 + r;
            uint4 v = *e;
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = pack_bf16x2(bf16_to_f32((uint16_t)(w[j] & 0xffffu)) * by, bf16_to_f32((uint16_t)(w[j] >> 16)) * by);
            *e = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    part[g][r] = sum;
    __syncthreads();
    if (g == 0) {
        const float by = before == c ? 1.f : __builtin_amdgcn_exp2f(before - c);
        sum = held * by;
#pragma unroll
        for (int i = 0; i < 64; ++i) sum += part[i][r];
        total[row] = sum;
        shift[row] = c;
        factor[row] = by;
    }
}

// ------------------------------------------------------------------------- the second product
struct ProductParams {
    const void *b;             // KT: [depth, cols], else its transpose
    int64_t ld, depth, cols;
    bool kt;
    const uint4 *packed;       // [rows, depth]
    int64_t blocks, b_apart, packed_apart;   // units between two terms
    int64_t np, nl;
    int64_t rows;
    void *out;
    int64_t ldo, slab;         // elements between two splits' outputs
    int steps_per_split, steps;
    const float *factor;       // per row: out = factor out + sum; null: out = sum
    int vec;
};

// out[row, col] (= factor out +) sum_k packed(row, k) b(k, col), one split of the reduction per y, each
// with an output of its own, and an XCD with all tiles of a split (one row x 49152 x 2048: 34 us, 46 where a
// split's tiles were spread over the XCDs). Splits fill the compute units where the tiles alone do not (splits_for);
// equal shares of all tiles' steps for each workgroup, which leave none idle, cost more than that: their
// workgroups no longer read the same part of the head at once (2665 rows x 49152 x 2048, 11 x 8 tiles:
// the whole call 1.10 ms with splits, 1.29 with shares). 4001 rows x 49152 x 2048: 623 us, 1.29 PFLOP/s.
template <int WP, int WL, int PF, int LF, bool KT, int OUT, int TERMS>
__global__ __launch_bounds__(64 * WP * WL) void product_kernel(const ProductParams p) {
    using C = Core<WP, WL, PF, LF, KT, true, TERMS>;
    __shared__ uint4 stages[3 * C::kStage];
    // an XCD takes all tiles of the same splits, which share what they read (257 rows x 32003 x 1000 with both
    // gradients 220 us, 232 with a split's tiles spread over the XCDs)
    const int64_t tiles = p.np * p.nl, t = by_xcd(blockIdx.x + tiles * blockIdx.y, tiles * gridDim.y);
    const int split = (int)(t / tiles);
    int64_t tp, tl;
    tile_at(t - split * tiles, p.np, p.nl, tp, tl);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wp = wave % WP, wl = wave / WP, q = lane >> 4;
    const int beg = split * p.steps_per_split;
    const int end = beg + p.steps_per_split < p.steps ? beg + p.steps_per_split : p.steps;
    // the split's own range of the staged operand, so that offsets stay within 32 bits
    C core;
    const int64_t k0 = (int64_t)beg * kStep;
    const int64_t depth = (end < p.steps ? (int64_t)end * kStep : p.depth) - k0;   // none: an empty split
    core.init(static_cast<const char *>(p.b) + (KT ? k0 * p.ld + tl * C::BL : tl * C::BL * p.ld + k0) * C::ES, p.ld, p.cols - tl * C::BL, depth,
              p.packed + (int64_t)beg * 128, tp * (C::BP / 16), p.blocks, wave);
    if constexpr (TERMS > 1) core.terms(p.b_apart, p.packed_apart);
    f32x4 acc[LF][PF];
    core.run(stages, acc);
#pragma unroll
    for (int j = 0; j < PF; ++j) {
        const int64_t row = tp * C::BP + (wp * PF + j) * 16 + (lane & 15);
        if (row >= p.rows) continue;
        const float factor = p.factor ? p.factor[row] : 0.f;
#pragma unroll
        for (int f = 0; f < LF; ++f) {
            const int64_t col = tl * C::BL + (wl * LF + f) * 16 + 4 * q;
            if (col >= p.cols) continue;
            f32x4 v = acc[f][j];
            if constexpr (OUT == CT_F32) {
                float *o = static_cast<float *>(p.out) + split * p.slab + row * p.ldo + col;
                if (p.vec && col + 4 <= p.cols) {
                    if (p.factor) {
                        const float4 old = *reinterpret_cast<const float4 *>(o);
                        v[0] += factor * old.x;
                        v[1] += factor * old.y;
                        v[2] += factor * old.z;
                        v[3] += factor * old.w;
                    }
                    *reinterpret_cast<float4 *>(o) = make_float4(v[0], v[1], v[2], v[3]);
                } else {
                    for (int i = 0; i < 4; ++i)
                        if (col + i < p.cols) o[i] = p.factor ? v[i] + factor * o[i] : v[i];
                }
            } else {
                uint16_t *o = static_cast<uint16_t *>(p.out) + row * p.ldo + col;
                if (p.vec && col + 4 <= p.cols) {
                    *reinterpret_cast<uint2 *>(o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
                } else {
                    for (int i = 0; i < 4; ++i)
                        if (col + i < p.cols) o[i] = bf16_bits(v[i]);
                }
            }
        }
    }
}

// ------------------------------------------------------------------------- logits in memory
struct RowParams {
    float *logits;             // [chunks][rows][vocab], summed into the first
    int chunks;
    int64_t slab, rows, vocab;
    float scale;
    float *shift, *total;
    const int *index;
    const uint16_t *first;
    float *chosen;
    int entries;
    int64_t units;
    uint4 *piece;
    int64_t piece_blocks, piece_apart;
    const float *near, *factor, *inverse;
};

// What logits_kernel<EXP> and join_kernel do, a workgroup per row; zeros past the vocabulary up to a
// whole step of the product that follows. TERMS 0: the statistics alone.
template <int TERMS>
__global__ __launch_bounds__(256) void rows_exp(const RowParams p) {
    __shared__ float lds[256];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    float *l = p.logits + row * p.vocab;
    float top = -INFINITY;
    for (int64_t v = tid; v < p.vocab; v += 256) {
        float x = l[v];
        for (int s = 1; s < p.chunks; ++s) x += l[s * p.slab + v];
        l[v] = x;
        top = fmaxf(top, x);
    }
    top = block_max<256>(top, lds);
    const float c = fmaxf(ceilf(top * p.scale), kNone);
    const int n = p.first[row * (p.units + 1) + p.units];
    for (int e = tid; e < n; e += 256) {
        float *at = l + p.index[row * p.entries + e];
        p.chosen[row * p.entries + e] = *at;
        *at = -INFINITY;
    }
    __syncthreads();
    float sum = 0.f;
    for (int64_t u = tid; u < up(p.vocab, kStep) / 8; u += 256) {   // 32 entries: four units
        const int64_t block = u >> 2;
        const int q = (int)(u & 3);
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t v = block * 32 + (i >> 2) * 16 + q * 4 + (i & 3);
            e[i] = v < p.vocab ? __builtin_amdgcn_exp2f(__builtin_fmaf(l[v], p.scale, -c)) : 0.f;
            sum += e[i];
        }
        if constexpr (TERMS > 0)
            store_unit<TERMS>(p.piece + ((row >> 4) * p.piece_blocks + block) * 64 + q * 16 + (row & 15), p.piece_apart, e);
    }
    sum = block_sum<256>(sum, lds);
    if (tid == 0) {
        p.shift[row] = c;
        p.total[row] = sum;
    }
}

// What logits_kernel<GRAD> does, a workgroup per row; zeros in the rows of the padding.
template <int TERMS>
__global__ __launch_bounds__(256) void rows_grad(const RowParams p) {
    const int64_t row = blockIdx.x;
    const int in = (int)(row & 31);
    uint16_t *out = reinterpret_cast<uint16_t *>(p.piece) +
                    ((row >> 5) * 64 + (in & 15) / 4 * 16) * 8 + (in & 3) + (in >> 4) * 4;
    const auto put = [&](int64_t v, float d) {
#pragma unroll
        for (int s = 0; s < TERMS; ++s) {
            const uint16_t bits = bf16_bits(d);
            out[s * p.piece_apart * 8 + ((v >> 4) * p.piece_blocks * 64 + (v & 15)) * 8] = bits;
            d -= bf16_to_f32(bits);
        }
    };
    if (row >= p.rows) {
        for (int64_t v = threadIdx.x; v < p.vocab; v += 256) put(v, 0.f);
        return;
    }
    const float *l = p.logits + row * p.vocab;
    const float c = p.near[row], f = p.factor[row];
    for (int64_t v = threadIdx.x; v < p.vocab; v += 256) {
        float x = l[v];
        for (int s = 1; s < p.chunks; ++s) x += l[s * p.slab + v];
        put(v, __builtin_amdgcn_exp2f(__builtin_fmaf(x, p.scale, -c)) * f);
    }
    __syncthreads();
    const int n = p.first[row * (p.units + 1) + p.units];
    for (int e = (int)threadIdx.x; e < n; e += 256)
        put(p.index[row * p.entries + e], p.inverse[row] * p.chosen[row * p.entries + e]);
}

// ------------------------------------------------------------------------- the ends
// A row's loss, the coefficients Q p_k - q_k of its targets in place of their logits, and Z with the
// targets' own terms in place of the others' sum. In double, from the targets' exponentials and the
// others' sum: log p_k = -log1p((Z - e_k) / e_k), Q p_k - q_k = (Q - q_k) - Q (Z - e_k) / Z.
__global__ __launch_bounds__(64) void row_loss(const float *__restrict__ shift, float *__restrict__ total,
                                               const float *__restrict__ weight, const float *__restrict__ mass,
                                               const float *__restrict__ entropy, const int *__restrict__ index,
                                               const float *__restrict__ q, float *__restrict__ chosen, int64_t rows,
                                               int entries, double inverse_t, int hard, double *__restrict__ losses) {
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x;
    const double c = shift[row], others = total[row], held = mass[row], ln2 = 0.693147180559945309417;
    const auto exponent = [&](int64_t at) { return (double)chosen[at] * inverse_t - c * ln2; };
    double own = 0;
    for (int e = lane; e < entries; e += 64)
        if (index[row * entries + e] != kNoEntry) own += exp(exponent(row * entries + e));
    for (int o = 32; o > 0; o >>= 1) own += __shfl_xor(own, o, 64);
    const double z = others + own;
    double sum = 0;
    for (int e = lane; e < entries; e += 64) {
        const int64_t at = row * entries + e;
        const double qk = q[at];
        if (index[at] == kNoEntry) {
            if (hard) sum += log(z) + c * ln2;   // a label outside the vocabulary: the row's loss is log Z
            chosen[at] = 0.f;
            continue;
        }
        const double x = exponent(at), ek = exp(x);
        // exact where the row has one target, which `own` then is
        const double rest = entries == 1 || own == ek ? others : others + (own - ek);
        if (qk != 0.0) sum += qk * (ek > 0 ? log1p(rest / ek) : log(z) - x);
        chosen[at] = (float)((held - qk) - held * (rest / z));
    }
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
    if (lane == 0) {
        losses[row] = held == 0.0 && !hard ? 0.0 : (double)weight[row] * (sum + (double)entropy[row]);
        total[row] = (float)z;
    }
}

__global__ __launch_bounds__(1024) void total_loss(const double *__restrict__ losses, int64_t rows, float *__restrict__ loss) {
    __shared__ double lds[1024];
    double sum = 0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) sum += losses[i];
    lds[threadIdx.x] = sum;
    __syncthreads();
    for (int h = 512; h > 0; h >>= 1) {
        if (threadIdx.x < h) lds[threadIdx.x] += lds[threadIdx.x + h];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = (float)lds[0];
}

// What the derivative of a row is made with, 0 in the padding: inverse = c_i u / T, and
// near + log2 of (factor / inverse) = log2 (Q_i / Z_i) with a whole number `near` as close to log2 Z_i
// as that allows, so that probabilities down to 2^-126 are held.
__global__ __launch_bounds__(256) void row_factors(const float *__restrict__ weight, const float *__restrict__ mass,
                                                   const float *__restrict__ shift, const float *__restrict__ total,
                                                   const float *__restrict__ upstream, float inverse_t, int64_t rows,
                                                   int64_t rows_pad, float *__restrict__ near, float *__restrict__ factor,
                                                   float *__restrict__ inverse) {
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= rows_pad) return;
    const float f = row < rows ? weight[row] * *upstream * inverse_t : 0.f;
    int size = 0;
    const float z = frexpf(total[row], &size);
    inverse[row] = f;
    near[row] = shift[row] + (float)size;
    factor[row] = row < rows && mass[row] != 0.f ? f * mass[row] / z : 0.f;
}

// dh_i = u c_i / T (Q_i / Z_i sums_i + sum_k coefficient_k w_v_k), times how often the row is given: rows of one
// number are equal, and each of them writes that value. A wave takes a row and 512 columns,
// four waves of a workgroup 2048; where there are many splits or targets (SHARE) the four take the
// same 512 columns, every fourth split and target each, and are joined in order. Bound by the sums and
// by the targets' rows of the head, K x width per row of the loss, from the caches (8192 rows of 64 x
// 2048: 255 us, 8.4 TB/s).
template <int IN, int OUT, bool VEC, bool SHARE>
__global__ __launch_bounds__(256) void hidden_grad_kernel(const float *__restrict__ sums, int splits, int64_t slab,
                                                          int64_t width, const float *__restrict__ weight,
                                                          const float *__restrict__ mass, const float *__restrict__ total,
                                                          const float *__restrict__ upstream, float inverse_t,
                                                          const int *__restrict__ index,
                                                          const float *__restrict__ coefficient, int entries,
                                                          const void *__restrict__ head, int64_t ld,
                                                          const int64_t *__restrict__ rows, int64_t tokens,
                                                          void *__restrict__ out, int64_t ldo, int64_t out_width, int whole,
                                                          const Repeats repeats) {
    __shared__ float lds[SHARE ? 4 : 1][512];
    const int64_t row = blockIdx.x, to = rows ? rows[row] : row;
    if (to < 0 || to >= tokens) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const float times = repeats.slots ? (float)repeats.slots[repeats.size + repeats.place[row]] : 1.f;
    const float held = mass[row], f = weight[row] * *upstream * inverse_t * times;
    const float by = held != 0.f ? held / total[row] : 0.f;
    const int64_t c0 = ((int64_t)blockIdx.y * (SHARE ? 1 : 4) + (SHARE ? 0 : wave)) * 512 + lane * 8;
    constexpr int STEP = SHARE ? 4 : 1;
    const int start = SHARE ? wave : 0;
    const auto in = [&](int i) { return VEC ? c0 < width : c0 + i < width; };
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = start; s < splits; s += STEP) {
        const float *p = sums + s * slab + row * width + c0;
        if constexpr (VEC) {
            if (in(0)) {
                const float4 x = *reinterpret_cast<const float4 *>(p), y = *reinterpret_cast<const float4 *>(p + 4);
                v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w, v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (in(i)) v[i] += p[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= by;
    const int *at = index + row * entries;
    const float *k = coefficient + row * entries;
#pragma unroll 8
    for (int e = start; e < entries; e += STEP) {
        const int vocab = at[e];
        if (vocab == kNoEntry) continue;
        const float by_k = k[e];
        if constexpr (IN == CT_F32) {
            const float *w = static_cast<const float *>(head) + vocab * ld + c0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (VEC ? c0 < width : c0 + i < width) v[i] += by_k * w[i];
        } else if (in(0)) {   // rows of whole units
            const uint4 x = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(head) + vocab * ld + c0);
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] += by_k * bf16_to_f32((uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu));
        }
    }
    if constexpr (!SHARE) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = held != 0.f ? v[i] * f : 0.f;
        if (OUT == CT_BF16 && whole && c0 + 8 <= out_width) {
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(out) + to * ldo + c0) = make_uint4(
                pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]), pack_bf16x2(o[4], o[5]), pack_bf16x2(o[6], o[7]));
            return;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (c0 + i >= out_width) continue;
            if constexpr (OUT == CT_F32) static_cast<float *>(out)[to * ldo + c0 + i] = o[i];
            else static_cast<uint16_t *>(out)[to * ldo + c0 + i] = bf16_bits(o[i]);
        }
        return;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) lds[wave][lane * 8 + i] = v[i];
        __syncthreads();
        for (int c = threadIdx.x; c < 512; c += 256) {
            const int64_t col = (int64_t)blockIdx.y * 512 + c;
            if (col >= out_width) break;
            const float sum = held != 0.f ? (lds[0][c] + lds[1][c] + lds[2][c] + lds[3][c]) * f : 0.f;
            if constexpr (OUT == CT_F32) static_cast<float *>(out)[to * ldo + col] = sum;
            else static_cast<uint16_t *>(out)[to * ldo + col] = bf16_bits(sum);
        }
    }
}

// The term arrays of float32 rows lie `terms_apart` 16-byte units apart.
hipError_t transpose(const void *x, int dtype, int64_t ld, int64_t rows, int64_t cols, void *out, int64_t pitch,
                     hipStream_t s) {
    const dim3 grid((unsigned)cdiv(rows, 64), (unsigned)cdiv(cols, 64));
    uint4 *to = static_cast<uint4 *>(out);
    if (dtype == CT_F32)
        transpose_rows<<<grid, dim3(256), 0, s>>>(static_cast<const float *>(x), ld, rows, cols, to, pitch, cols * pitch / 8);
    else
        transpose_rows<<<grid, dim3(256), 0, s>>>(static_cast<const uint16_t *>(x), ld, rows, cols, to, pitch, (int64_t)0);
    return hipGetLastError();
}

template <class T>
T *at(void *base, int64_t offset) {
    return reinterpret_cast<T *>(static_cast<char *>(base) + offset);
}

template <int MODE, int TERMS>
hipError_t launch_logits(const Plan &pl, const LogitsParams &p, hipStream_t s) {
    const dim3 grid((unsigned)(p.np * p.nl));
    if (pl.bp == 64) logits_kernel<4, 1, 1, 8, MODE, TERMS><<<grid, dim3(256), 0, s>>>(p);
    if constexpr (TERMS != 3)   // float32 has the narrow tile there
        if (pl.bp == 128) logits_kernel<8, 1, 1, 16, MODE, TERMS><<<grid, dim3(512), 0, s>>>(p);
    if constexpr (MODE == GRAD || TERMS != 2)   // E of so many rows is one term or three
        if (pl.bp == 256) logits_kernel<8, 1, 2, 16, MODE, TERMS><<<grid, dim3(512), 0, s>>>(p);
    return hipGetLastError();
}
template <int MODE>
hipError_t launch_logits(const Plan &pl, const LogitsParams &p, hipStream_t s) {
    if (pl.tri) return launch_logits<MODE, 3>(pl, p, s);
    if constexpr (MODE != STATS)
        if (pl.terms[MODE] == 2) return launch_logits<MODE, 2>(pl, p, s);
    return launch_logits<MODE, 1>(pl, p, s);
}
template <int OUT, bool KT, int TERMS>
hipError_t launch_product(int bp, const ProductParams &p, int splits, hipStream_t s) {
    const dim3 grid((unsigned)(p.np * p.nl), (unsigned)splits);
    if (bp == 64) {
        if constexpr (KT || (OUT == CT_F32 && TERMS != 2))
            product_kernel<4, 1, 1, 8, KT, OUT, TERMS><<<grid, dim3(256), 0, s>>>(p);
    } else if (bp == 128) {
        if constexpr (TERMS < 3) product_kernel<8, 1, 1, 16, KT, OUT, TERMS><<<grid, dim3(512), 0, s>>>(p);
    } else {
        if constexpr (!KT && TERMS != 2) product_kernel<8, 1, 2, 16, false, OUT, TERMS><<<grid, dim3(512), 0, s>>>(p);
    }
    return hipGetLastError();
}
// Packed operands of two terms take the narrower tiles: the wider ones have no registers for them.
template <int OUT>
hipError_t launch_product(int bp, int terms, const ProductParams &p, int splits, hipStream_t s) {
    if constexpr (OUT == CT_F32)
        if (terms == 3)
            return p.kt ? launch_product<OUT, true, 3>(bp, p, splits, s) : launch_product<OUT, false, 3>(bp, p, splits, s);
    if (p.kt) return terms == 2 ? launch_product<OUT, true, 2>(bp, p, splits, s) : launch_product<OUT, true, 1>(bp, p, splits, s);
    return terms == 2 ? launch_product<OUT, false, 2>(bp, p, splits, s) : launch_product<OUT, false, 1>(bp, p, splits, s);
}

// hidden: the hidden rows are read (in a backward, for the head's gradient). forward: the targets are read
// from the tables; later they are in what is kept.
int check(const ct_head_loss *a, bool hidden, bool forward) {
    if (!a) return -CT_EINVAL_POINTER;
    if (a->dtype != CT_BF16 && a->dtype != CT_F32) return -CT_EINVAL_DTYPE;
    if (a->count < 0 || a->count > kMaxRows || a->width <= 0 || a->width > kMaxWidth || a->vocab <= 0 ||
        a->vocab > kMaxVocab || a->entries < 1 || a->entries > kMaxEntries)
        return -CT_EINVAL_SHAPE;
    if (a->tokens < 0 || (!a->rows && a->tokens < a->count)) return -CT_EINVAL_SHAPE;
    if (a->hidden_width <= 0 || a->hidden_width > a->width || a->ld_hidden < a->hidden_width || a->ld_head < a->width ||
        a->ld_hidden > kMaxPitch || a->ld_head > kMaxPitch)
        return -CT_EINVAL_SHAPE;
    if (a->count && forward && !a->values && a->entries != 1) return -CT_EINVAL_SHAPE;   // empty tables have no address
    if (forward && (a->ld_indices < a->entries || (a->values && a->ld_values < a->entries))) return -CT_EINVAL_SHAPE;
    if (up(a->count, 256) * up(a->width, kStep) > kMaxValues) return -CT_EINVAL_SHAPE;
    if (!forward && hidden && a->count > kMaxHeadRows) return -CT_EINVAL_SHAPE;
    if (!(a->temperature > 0)) return -CT_EINVAL_SHAPE;
    if (a->count && ((hidden && !a->hidden) || !a->head)) return -CT_EINVAL_POINTER;
    if (a->count && forward && (!a->indices || !a->weights)) return -CT_EINVAL_POINTER;
    if (a->dtype == CT_BF16 && (a->width % 8 || a->ld_head % 8)) return -CT_EINVAL_SHAPE;
    if (a->dtype == CT_BF16 && reinterpret_cast<uintptr_t>(a->head) % 16) return -CT_EINVAL_POINTER;
    return 0;
}
Source source(const ct_head_loss *a) { return Source{a->hidden, a->rows, a->ld_hidden, a->count, a->tokens, a->hidden_width}; }
// Whether the hidden rows can be read as they lie: [count, width] rows, for bf16 in 16-byte units.
bool in_place(const ct_head_loss *a) {
    if (a->rows || a->hidden_width != a->width) return false;
    return a->dtype == CT_F32 || (a->ld_hidden % 8 == 0 && reinterpret_cast<uintptr_t>(a->hidden) % 16 == 0);
}
int check_sizes(int64_t count, int64_t width, int64_t vocab, int32_t entries, int32_t dtype) {
    if (dtype != CT_BF16 && dtype != CT_F32) return -CT_EINVAL_DTYPE;
    return count < 0 || count > kMaxRows || width <= 0 || width > kMaxWidth || vocab <= 0 || vocab > kMaxVocab ||
                   entries < 1 || entries > kMaxEntries || up(count, 256) * up(width, kStep) > kMaxValues
               ? -CT_EINVAL_SHAPE
               : 0;
}
#define CT_TRY(call)                            \
    do {                                        \
        const hipError_t e_ = (call);           \
        if (e_ != hipSuccess) return (int)e_;   \
    } while (0)

LogitsParams logits_params(const ct_head_loss *a, const Plan &pl, const Kept &k, const Scratch &sc, void *kept, void *ws) {
    LogitsParams p{};
    p.ld = pl.tri && pl.turned ? up(pl.width, 8) : a->ld_head;
    p.width = pl.tri && !pl.turned ? pl.width : up(pl.width, 8);
    p.head_apart = pl.piece * p.ld / 8;
    p.packed_apart = pl.rows_pad * pl.width_pad / 8;
    p.piece_apart = pl.rows_pad * pl.piece / 8;
    p.packed = at<const uint4>(ws, sc.packed);
    p.blocks = pl.width_pad / 32;
    p.np = pl.rows_pad / pl.bp;
    p.scale = (float)(1.4426950408889634074 / a->temperature);
    p.piece = at<uint4>(ws, sc.piece);
    p.stats = at<float2>(ws, sc.stats);
    p.rows_pad = pl.rows_pad;
    p.rows = pl.rows;
    p.index = at<int>(kept, k.index);
    p.first = at<uint16_t>(kept, k.first);
    p.chosen = at<float>(kept, k.chosen);
    p.entries = (int)pl.entries;
    p.units = pl.units;
    return p;
}

// The logits of the whole vocabulary in memory, in chunks of their reduction, and the row pass's operands.
hipError_t logits_in_memory(const Plan &pl, const LogitsParams &p, void *ws, const Scratch &sc, RowParams &r, hipStream_t s) {
    ProductParams g{};
    g.b = p.head;
    g.ld = p.ld;
    g.depth = p.width;
    g.cols = pl.vocab;
    g.packed = p.packed;
    g.blocks = p.blocks;
    g.b_apart = p.head_apart;
    g.packed_apart = p.packed_apart;
    g.np = p.np;
    g.nl = cdiv(pl.vocab, pl.bl);
    g.rows = pl.rows;
    g.out = at<float>(ws, sc.logits);
    g.ldo = pl.vocab;
    g.slab = pl.rows * pl.vocab;
    g.steps = (int)cdiv(p.width, kStep);
    g.steps_per_split = (int)cdiv(g.steps, pl.chunks);
    g.vec = pl.vocab % 4 == 0;
    r.logits = at<float>(ws, sc.logits);
    r.chunks = pl.chunks;
    r.slab = g.slab;
    r.rows = pl.rows;
    r.vocab = pl.vocab;
    r.scale = p.scale;
    r.index = p.index;
    r.first = p.first;
    r.chosen = p.chosen;
    r.entries = p.entries;
    r.units = p.units;
    r.piece = p.piece;
    r.piece_blocks = p.piece_blocks;
    r.piece_apart = p.piece_apart;
    return launch_product<CT_F32>(pl.bp, pl.tri ? 3 : 1, g, pl.chunks, s);
}

Repeats repeats_of(const ct_head_loss *a, const Plan &pl, const Kept &k, void *kept, bool hidden_grad) {
    if (!a->rows || !hidden_grad) return Repeats{nullptr, nullptr, 0};
    return Repeats{at<int>(kept, k.slots), at<int>(kept, k.place), slots_for(pl.rows)};
}

hipError_t pack_hidden(const ct_head_loss *a, const Plan &pl, void *packed, const Repeats &cleared, hipStream_t stream) {
    const int64_t units = pl.rows_pad / 16 * (pl.width_pad / 32) * 64;
    const Source src = source(a);
    if (pl.tri) {
        pack_split<<<dim3((unsigned)cdiv(units, 256)), dim3(256), 0, stream>>>(src, pl.width_pad / 32,
                                                                              static_cast<uint4 *>(packed), units, cleared);
        return hipGetLastError();
    }
    const bool vec = a->hidden_width % 8 == 0 && a->ld_hidden % 8 == 0 && reinterpret_cast<uintptr_t>(a->hidden) % 16 == 0;
    const dim3 grid((unsigned)cdiv(units, 256));
    if (vec) pack_rows<true><<<grid, dim3(256), 0, stream>>>(src, pl.width_pad / 32, static_cast<uint4 *>(packed), units, cleared);
    else pack_rows<false><<<grid, dim3(256), 0, stream>>>(src, pl.width_pad / 32, static_cast<uint4 *>(packed), units, cleared);
    return hipGetLastError();
}
hipError_t split_terms(const float *x, int64_t ld, int64_t rows, int64_t cols, uint4 *out, int64_t pitch, int64_t apart,
                       hipStream_t s) {
    const dim3 grid((unsigned)cdiv(rows * (pitch / 8), 256));
    const bool pairs = ld % 2 == 0 && reinterpret_cast<uintptr_t>(x) % 8 == 0;
    if (pairs) split_rows<true><<<grid, dim3(256), 0, s>>>(x, ld, rows, cols, out, pitch, apart);
    else split_rows<false><<<grid, dim3(256), 0, s>>>(x, ld, rows, cols, out, pitch, apart);
    return hipGetLastError();
}
// The piece of the head that starts at entry v0, as the logits kernel stages it: in place, or on the
// wide tiles float32 rows in their three terms.
hipError_t head_piece(const ct_head_loss *a, const Plan &pl, LogitsParams &p, int64_t v0, int64_t cols, void *split,
                      hipStream_t stream) {
    p.v0 = v0;
    p.v1 = v0 + cols;
    p.nl = cdiv(cols, pl.bl);
    if (!pl.tri || !pl.turned) {
        p.head = static_cast<const char *>(a->head) + v0 * a->ld_head * (pl.tri ? 4 : 2);
        return hipSuccess;
    }
    p.head = split;
    return split_terms(static_cast<const float *>(a->head) + v0 * a->ld_head, a->ld_head, cols, pl.width,
                       static_cast<uint4 *>(split), p.ld, p.head_apart, stream);
}
// The loss's rows one after the other: as they lie, or gathered into `to`.
hipError_t plain_hidden(const ct_head_loss *a, const Plan &pl, void *to, const void **hidden, int64_t *ld, hipStream_t stream) {
    if (in_place(a)) {
        *hidden = a->hidden;
        *ld = a->ld_hidden;
        return hipSuccess;
    }
    *hidden = to;
    *ld = pl.width;
    const dim3 grid((unsigned)pl.rows);
    if (a->dtype == CT_F32) gather_rows<float><<<grid, dim3(256), 0, stream>>>(source(a), static_cast<float *>(to), pl.width);
    else gather_rows<uint16_t><<<grid, dim3(256), 0, stream>>>(source(a), static_cast<uint16_t *>(to), pl.width);
    return hipGetLastError();
}

}  // namespace
}  // namespace ct

using namespace ct;

extern "C" int64_t ct_head_loss_kept(int64_t count, int64_t width, int64_t vocab, int32_t entries, int32_t dtype,
                                     int32_t hidden_grad) {
    if (check_sizes(count, width, vocab, entries, dtype) || count == 0) return 0;
    return kept_of(plan_of(count, width, vocab, entries, dtype), hidden_grad != 0).bytes;
}

extern "C" int64_t ct_head_loss_workspace(int64_t count, int64_t width, int64_t vocab, int32_t entries, int32_t dtype,
                                          int32_t pass) {
    if (check_sizes(count, width, vocab, entries, dtype) || count == 0 || pass < 0 || pass > 2 ||
        (pass == 2 && count > kMaxHeadRows))
        return 0;
    return scratch_of(plan_of(count, width, vocab, entries, dtype), pass).bytes;
}

extern "C" int ct_head_loss_forward(const ct_head_loss *a, float *loss, int32_t hidden_grad, void *kept,
                                    int64_t kept_bytes, void *workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (const int bad = check(a, true, true)) return bad;
    if (!loss) return -CT_EINVAL_POINTER;
    if (a->count == 0) {
        total_loss<<<dim3(1), dim3(1024), 0, stream>>>(nullptr, 0, loss);
        return (int)hipGetLastError();
    }
    const Plan pl = plan_of(a->count, a->width, a->vocab, a->entries, a->dtype);
    const Kept k = kept_of(pl, hidden_grad != 0);
    const Scratch sc = scratch_of(pl, hidden_grad ? 1 : 0);
    if (!kept || kept_bytes < k.bytes || !workspace || workspace_bytes < sc.bytes ||
        reinterpret_cast<uintptr_t>(kept) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16)
        return -CT_EINVAL_WORKSPACE;
    const double inverse_t = 1.0 / a->temperature;
    float *shift = at<float>(kept, k.shift), *total = at<float>(kept, k.total), *sums = at<float>(kept, k.sums);
    float *factor = at<float>(workspace, sc.factor);
    const Targets t{a->rows, a->tokens, a->indices, a->values, a->log_normalizer, a->weights, a->ld_indices, a->ld_values};
    const Repeats repeats = repeats_of(a, pl, k, kept, hidden_grad != 0);
    const auto targets = [&](auto kernel, int threads) {
        kernel<<<dim3((unsigned)pl.rows_pad), dim3(threads), 0, stream>>>(
            t, pl.rows, (int)pl.entries, pl.vocab, pl.units, inverse_t, at<int>(kept, k.index), at<float>(kept, k.q),
            at<float>(kept, k.chosen), at<uint16_t>(kept, k.first), at<float>(kept, k.weight), at<float>(kept, k.mass),
            at<float>(kept, k.entropy), shift, total, repeats);
    };
    // Numbered rows are packed first, which clears their slots. Others last: the first launch of a pass waits for
    // what it reads, longer for the hidden rows than for the tables (one row: 2 us).
    if (repeats.slots) CT_TRY(pack_hidden(a, pl, at<void>(workspace, sc.packed), repeats, stream));
    if (pl.entries <= 64) targets(targets_kernel<64, 64>, 64);
    else targets(targets_kernel<256, kMaxEntries>, 256);
    CT_TRY(hipGetLastError());
    if (!repeats.slots) CT_TRY(pack_hidden(a, pl, at<void>(workspace, sc.packed), repeats, stream));

    LogitsParams p = logits_params(a, pl, k, sc, kept, workspace);
    const int64_t piece = sweep_piece(pl, hidden_grad ? 1 : 0);
    for (int64_t v0 = 0; v0 < pl.vocab; v0 += piece) {
        const int64_t cols = pl.vocab - v0 < piece ? pl.vocab - v0 : piece;
        CT_TRY(head_piece(a, pl, p, v0, cols, at<void>(workspace, sc.split), stream));
        p.piece_blocks = pl.piece / 32;
        if (pl.chunks > 1) {
            RowParams r{};
            CT_TRY(logits_in_memory(pl, p, workspace, sc, r, stream));
            r.shift = shift;
            r.total = total;
            const dim3 grid((unsigned)pl.rows);
            const int terms = hidden_grad ? pl.terms[1] : 0;
            if (terms == 0) rows_exp<0><<<grid, dim3(256), 0, stream>>>(r);
            else if (terms == 1) rows_exp<1><<<grid, dim3(256), 0, stream>>>(r);
            else if (terms == 2) rows_exp<2><<<grid, dim3(256), 0, stream>>>(r);
            else rows_exp<3><<<grid, dim3(256), 0, stream>>>(r);
        } else {
            CT_TRY(hidden_grad ? launch_logits<EXP>(pl, p, stream) : launch_logits<STATS>(pl, p, stream));
            join_kernel<<<dim3((unsigned)(pl.rows_pad / 16)), dim3(1024), 0, stream>>>(
                p.stats, (int)cdiv(cols, kUnit), pl.rows_pad, shift, total, factor, hidden_grad ? p.piece : nullptr,
                p.piece_blocks, pl.terms[hidden_grad ? 1 : 0], p.piece_apart);
        }
        CT_TRY(hipGetLastError());
        if (!hidden_grad) continue;
        ProductParams g{};
        g.b = p.head;
        g.ld = p.ld;
        g.kt = !pl.turned;
        if (pl.turned) {
            uint16_t *turned = at<uint16_t>(workspace, sc.turned);
            const void *from = static_cast<const char *>(a->head) + v0 * a->ld_head * (pl.tri ? 4 : 2);
            CT_TRY(transpose(from, pl.dtype, a->ld_head, cols, pl.width, turned, pl.piece, stream));
            g.b = turned;
            g.ld = pl.piece;
        }
        g.b_apart = pl.turned ? pl.width * pl.piece / 8 : p.head_apart;
        g.packed_apart = p.piece_apart;
        g.depth = pl.turned ? up(cols, kStep) : cols;   // turned rows end with a whole step, in their order
        g.cols = pl.width;
        g.packed = p.piece;
        g.blocks = p.piece_blocks;
        g.np = p.np;
        g.nl = cdiv(pl.width, pl.bl);
        g.rows = pl.rows;
        g.out = sums;
        g.ldo = pl.width;
        g.slab = pl.rows * pl.width;
        g.steps = (int)cdiv(cols, kStep);
        g.steps_per_split = (int)cdiv(g.steps, pl.splits);
        g.factor = v0 ? factor : nullptr;
        g.vec = pl.width % 4 == 0;
        CT_TRY(launch_product<CT_F32>(pl.bp, pl.terms[1], g, pl.splits, stream));
    }
    row_loss<<<dim3((unsigned)pl.rows), dim3(64), 0, stream>>>(
        shift, total, at<float>(kept, k.weight), at<float>(kept, k.mass), at<float>(kept, k.entropy),
        at<int>(kept, k.index), at<float>(kept, k.q), at<float>(kept, k.chosen), pl.rows, (int)pl.entries, inverse_t,
        a->values == nullptr, at<double>(workspace, sc.losses));
    CT_TRY(hipGetLastError());
    total_loss<<<dim3(1), dim3(1024), 0, stream>>>(at<double>(workspace, sc.losses), pl.rows, loss);
    return (int)hipGetLastError();
}

extern "C" int ct_head_loss_backward(const ct_head_loss *a, const float *upstream, const void *kept_in, int32_t hidden_grad,
                                     int64_t kept_bytes, void *d_hidden, int64_t ld_d_hidden, int64_t d_hidden_width,
                                     int32_t d_hidden_dtype, void *d_head, int64_t ld_d_head, int64_t d_head_width,
                                     int32_t d_head_dtype, void *workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (const int bad = check(a, d_head != nullptr, false)) return bad;
    if (a->count == 0) return 0;
    if (!upstream) return -CT_EINVAL_POINTER;
    const Plan pl = plan_of(a->count, a->width, a->vocab, a->entries, a->dtype);
    const Kept k = kept_of(pl, hidden_grad != 0);
    void *kept = const_cast<void *>(kept_in);
    if (!kept || kept_bytes < k.bytes || reinterpret_cast<uintptr_t>(kept) % 16) return -CT_EINVAL_WORKSPACE;
    const float inverse_t = (float)(1.0 / a->temperature);
    if (d_hidden) {
        if (!hidden_grad) return -CT_EINVAL_WORKSPACE;
        if (d_hidden_dtype != CT_F32 && d_hidden_dtype != CT_BF16) return -CT_EINVAL_DTYPE;
        if (d_hidden_width < 0 || d_hidden_width > pl.width || ld_d_hidden < d_hidden_width) return -CT_EINVAL_SHAPE;
        const bool share = pl.splits + pl.entries > 4, vec = pl.width % 8 == 0;
        const int whole = ld_d_hidden % 8 == 0 && reinterpret_cast<uintptr_t>(d_hidden) % 16 == 0;
        const auto run = [&](auto kernel) {
            kernel<<<dim3((unsigned)pl.rows, (unsigned)cdiv(d_hidden_width, share ? 512 : 2048)), dim3(256), 0, stream>>>(
                at<const float>(kept, k.sums), pl.splits, pl.rows * pl.width, pl.width, at<const float>(kept, k.weight),
                at<const float>(kept, k.mass), at<const float>(kept, k.total), upstream, inverse_t,
                at<const int>(kept, k.index), at<const float>(kept, k.chosen), (int)pl.entries, a->head, a->ld_head, a->rows,
                a->tokens, d_hidden, ld_d_hidden, d_hidden_width, whole, repeats_of(a, pl, k, kept, true));
        };
        const auto pick = [&](auto in, auto out, auto wide) {
            if (share) run(hidden_grad_kernel<decltype(in)::value, decltype(out)::value, decltype(wide)::value, true>);
            else run(hidden_grad_kernel<decltype(in)::value, decltype(out)::value, decltype(wide)::value, false>);
        };
        const std::integral_constant<int, CT_F32> f32;
        const std::integral_constant<int, CT_BF16> bf16;
        const std::true_type yes;
        const std::false_type no;
        const bool narrow = d_hidden_dtype == CT_BF16;
        if (pl.dtype == CT_BF16) narrow ? pick(bf16, bf16, yes) : pick(bf16, f32, yes);   // widths of whole units
        else if (vec) narrow ? pick(f32, bf16, yes) : pick(f32, f32, yes);
        else narrow ? pick(f32, bf16, no) : pick(f32, f32, no);
        CT_TRY(hipGetLastError());
    }
    if (!d_head) return 0;
    if (d_head_dtype != CT_F32 && d_head_dtype != CT_BF16) return -CT_EINVAL_DTYPE;
    if (pl.dtype == CT_F32 && d_head_dtype != CT_F32) return -CT_EINVAL_DTYPE;
    if (d_head_width < 0 || d_head_width > pl.width || ld_d_head < d_head_width) return -CT_EINVAL_SHAPE;
    const Scratch sc = scratch_of(pl, 2);
    if (!workspace || workspace_bytes < sc.bytes || reinterpret_cast<uintptr_t>(workspace) % 16) return -CT_EINVAL_WORKSPACE;
    float *factor = at<float>(workspace, sc.factor);
    float *inverse = at<float>(workspace, sc.inverse), *near = at<float>(workspace, sc.near);
    row_factors<<<dim3((unsigned)cdiv(pl.rows_pad, 256)), dim3(256), 0, stream>>>(
        at<const float>(kept, k.weight), at<const float>(kept, k.mass), at<const float>(kept, k.shift),
        at<const float>(kept, k.total), upstream, inverse_t, pl.rows, pl.rows_pad, near, factor, inverse);
    CT_TRY(hipGetLastError());
    CT_TRY(pack_hidden(a, pl, at<void>(workspace, sc.packed), Repeats{nullptr, nullptr, 0}, stream));
    const void *hidden;
    int64_t ld;
    CT_TRY(plain_hidden(a, pl, at<void>(workspace, sc.plain), &hidden, &ld, stream));
    LogitsParams p = logits_params(a, pl, k, sc, kept, workspace);
    p.shift = near;
    p.factor = factor;
    p.inverse = inverse;
    p.piece_blocks = pl.rows_pad / 32;
    int64_t apart = 0;
    if (pl.turned) {
        uint16_t *turned = at<uint16_t>(workspace, sc.turned);
        apart = pl.width * up(pl.rows, kStep) / 8;
        CT_TRY(transpose(hidden, pl.dtype, ld, pl.rows, pl.width, turned, up(pl.rows, kStep), stream));
        hidden = turned;
        ld = up(pl.rows, kStep);
    }
    for (int64_t v0 = 0; v0 < pl.vocab; v0 += pl.piece) {
        const int64_t cols = pl.vocab - v0 < pl.piece ? pl.vocab - v0 : pl.piece;
        CT_TRY(head_piece(a, pl, p, v0, cols, at<void>(workspace, sc.split), stream));
        if (pl.chunks > 1) {
            RowParams r{};
            CT_TRY(logits_in_memory(pl, p, workspace, sc, r, stream));
            r.near = near;
            r.factor = factor;
            r.inverse = inverse;
            const dim3 grid((unsigned)pl.rows_pad);
            if (pl.terms[2] == 1) rows_grad<1><<<grid, dim3(256), 0, stream>>>(r);
            else if (pl.terms[2] == 2) rows_grad<2><<<grid, dim3(256), 0, stream>>>(r);
            else rows_grad<3><<<grid, dim3(256), 0, stream>>>(r);
            CT_TRY(hipGetLastError());
        } else {
            CT_TRY(launch_logits<GRAD>(pl, p, stream));
        }
        ProductParams g{};
        g.b = hidden;
        g.ld = ld;
        g.kt = !pl.turned;
        g.b_apart = apart;
        g.packed_apart = p.piece_apart;
        g.depth = pl.turned ? up(pl.rows, kStep) : pl.rows;
        g.cols = d_head_width;
        g.packed = p.piece;
        g.blocks = p.piece_blocks;
        const int bp = pl.terms[2] == 2 && pl.bp == 256 ? 128 : pl.bp;
        g.np = cdiv(cols, bp);
        g.nl = cdiv(d_head_width, pl.bl);
        g.rows = cols;
        g.out = static_cast<char *>(d_head) + v0 * ld_d_head * (d_head_dtype == CT_F32 ? 4 : 2);
        g.ldo = ld_d_head;
        g.steps = g.steps_per_split = (int)cdiv(pl.rows, kStep);
        g.vec = ld_d_head % 4 == 0 && reinterpret_cast<uintptr_t>(d_head) % 16 == 0;
        CT_TRY(d_head_dtype == CT_F32 ? launch_product<CT_F32>(bp, pl.terms[2], g, 1, stream)
                                      : launch_product<CT_BF16>(bp, pl.terms[2], g, 1, stream));
    }
    return 0;
}
