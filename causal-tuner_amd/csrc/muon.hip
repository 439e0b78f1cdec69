// Orthogonalising matrices by Newton-Schulz products, and the Muon step around it, gfx950.
//
//   X_0 = M / max(|M|_F, eps);  X_{i+1} = a X_i + (b A_i + c A_i^2) X_i,  A_i = X_i X_i^T
//
// (short side first; M of more rows than columns is taken transposed). The iteration never
// leaves the span of powers of the short side's Gram matrix, so it runs there:
//   G_0 = X_0 X_0^T,  P_i = a I + b G_i + c G_i^2,  G_{i+1} = P_i G_i P_i,  X_n = P_{n-1} ... P_0 X_0
// (all of them symmetric and commuting). That takes one product to make G_0, r x r products,
// and one product with M, instead of two products with the whole matrix per step: for an
// adapter of rank 256 and width 4096 about a fifth of the operations.
//
// The Gram matrix squares the singular values, and a step multiplies the small ones by a =
// 3.4: with float32 sums in G the result was 5e-5 off at a spectrum over two decades and 1e-4
// over three (float32 steps on the whole matrix: 4e-6 and 6e-6). G, P and the products
// between them are therefore double (v_mfma_f64_16x16x4, which runs at half of float32's rate
// on a fifth of the work); only the last product, of the final P_{n-1} ... P_0 and M, is float32.
// Keeping P_{n-1} ... P_0 in float32 too would lose a factor of three in those cases.
//
// Every G is positive semidefinite, and G <- P G P keeps it so, but roundings of 1e-16 make the
// zero eigenvalues of a matrix of low rank negative. A step multiplies those by (a + b l + c l^2)^2,
// which grows with |l| where it falls for the positive ones: from 14 steps on (a^28 = 1e15) they
// ran away, at 20 the result was NaN. So each G gets gram_floor(r) = 2^-50 r on its diagonal, more
// than its roundings (2^-53 sqrt(r) times 40 at most: |P|^2 < 12, |G| < 1.5, two products) and less
// than shows: after 5 steps 1e-8 of what small singular values become. With it the result's error
// for a matrix of low rank is that of float32 steps on the whole matrix, since Q grows by a = 3.4 a
// step where M has nothing and its own rounding (2^-24) reaches M's rows: 2e-5 after 5 steps, 1e-2
// after 10, and a tenth from 14 on, where the floor ends Q's growth (float32 steps: 1 and more).
//
// What bounds it, two layers' adapters of rank 256 (36M elements, 749 us a step): the Gram
// pass 206 us (double matrix instructions, 70% of its cycles at a clock that they pull down to
// about 1.9 GHz; 12 bytes an element), the 14 launches of r x r products 22 us each (their
// operands' way from L2, half of it, and double matrix instructions, 45%), the last product 214 us
// (float32 matrix instructions, 62% of its cycles; 16 bytes an element, 2.7 TB/s, which alone
// take 170). Small sets: the launches. Whole models: every matrix has its own scratch, 949 MB for
// 24 layers of width 2048, and the launches go through it past the caches (338 us a layer, 264
// at 4 layers).
// Tried and left out: 64 x 64 tiles in the r x r products (the same at 24 matrices, 20% slower
// at 12), k-steps of 32 rows in flight instead of 16 (more registers, 3% slower).
//
// The Muon step (Jordan et al., Muon: an optimizer for hidden layers; torch.optim.Muon's
// arguments): m = mu m + (1 - mu) g, M = nesterov ? mu m + (1 - mu) g : m, and
// p = p (1 - lr decay) - lr adjust X_n, all matrices of one type in one set of launches.

#include <math.h>

#include <algorithm>
#include <vector>

#include "common.hpp"

namespace ct {
namespace {

typedef __attribute__((__vector_size__(4 * sizeof(double)))) double f64x4;
typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;

constexpr int kThreads = 256;
constexpr int kPad = 32;        // r x r matrices are stored with r rounded up to this
constexpr int kSmall = 64;      // short sides up to this iterate inside one workgroup
constexpr int kOnePass = 256;   // short sides up to this make their Gram matrix in one pass over M
constexpr int kGramTile = 64;   // rows of M per side of a Gram share past kOnePass
constexpr int kChunk = 32;      // long-side elements per LDS stage
constexpr int kEntry = 8;       // int32 per plan entry

struct Matrix {                 // ct_muon_matrix
    void *param;
    const void *grad;
    float *momentum;
    int64_t rows, cols;
    int64_t scratch;            // doubles from the workspace's start: the r x r buffers
    int64_t parts;              // and the partial Gram matrices
    float adjust;
    int32_t splits;             // partial Gram matrices
};

struct Item {
    int32_t matrix, i, j, lo, hi, slot, pad0, pad1;
};

struct Hyper {
    float lr, mu, rest, keep;   // rest = 1 - mu, keep = 1 - lr decay
    int nesterov, step;         // step: 0 = orthogonalize grad into param
    double a, b, c, eps;
};

// Pointers that come out of memory may be of any kind to the compiler, and its flat loads are
// waited for by every wait for LDS. These say that they are global: the Gram pass of two layers'
// adapters went from 250 us to 230 by that alone.
typedef float Float4 __attribute__((ext_vector_type(4)));
typedef uint32_t Uint2 __attribute__((ext_vector_type(2)));
template <typename V>
__device__ __forceinline__ V from_global(const void *p) {
    typedef const __attribute__((address_space(1))) V *Global;
    return *(Global)(uintptr_t)p;
}
template <typename V>
__device__ __forceinline__ void to_global(void *p, V v) {
    typedef __attribute__((address_space(1))) V *Global;
    *(Global)(uintptr_t)p = v;
}

__host__ __device__ __forceinline__ int64_t least(int64_t x, int64_t y) { return x < y ? x : y; }
__device__ __forceinline__ int short_side(const Matrix &m) { return (int)least(m.rows, m.cols); }
__host__ __device__ __forceinline__ int padded(int r) { return (r + kPad - 1) / kPad * kPad; }
__host__ __device__ __forceinline__ int tiles16(int r) { return (r + 15) / 16; }

// What every G has on its diagonal on top.
__device__ __forceinline__ double gram_floor(int r) { return padded(r) * 0x1p-50; }

// A partial Gram matrix: the squared norms of its part of M (one, or one per 64 rows), then
// the 16 x 16 tiles (i, j), i >= j, row by row.
__host__ __device__ __forceinline__ int part_head(int r) {
    return r <= kOnePass ? 2 : (r + kGramTile - 1) / kGramTile + 1 & ~1;
}
__host__ __device__ __forceinline__ int64_t part_size(int r) {
    const int64_t t = tiles16(r);
    return part_head(r) + t * (t + 1) / 2 * 256;
}
__device__ __forceinline__ double *part_of(const Matrix &m, double *ws, int slot) {
    return ws + m.parts + slot * part_size(short_side(m));
}
__device__ __forceinline__ int64_t tile_of(int i, int j) { return ((int64_t)i * (i + 1) / 2 + j) * 256; }

// The buffers of one matrix: 1 / |M|, then G, P, T and two Q (doubles; not for small ones)
// and the final float Q.
enum { kG = 0, kP = 1, kT = 2, kQ = 3, kBuffers = 5 };
__device__ __forceinline__ double *buffer(const Matrix &m, double *ws, int which) {
    const int64_t rp = padded(short_side(m));
    return ws + m.scratch + 2 + which * rp * rp;
}
__device__ __forceinline__ float *final_q(const Matrix &m, double *ws) {
    return reinterpret_cast<float *>(short_side(m) <= kSmall ? ws + m.scratch + 2 : buffer(m, ws, kBuffers));
}
// Element (row, k) of the final Q, ordered as the last product's lanes read it: lane (row, h)
// takes k = 8 s + 4 h .. + 3 in one 16-byte load, 64 lanes 1 KB in a row.
__device__ __forceinline__ int64_t final_at(int rp, int row, int k) {
    return (((int64_t)(k >> 3) * rp + row) * 2 + ((k >> 2) & 1)) * 4 + (k & 3);
}

template <typename T>
__device__ __forceinline__ float load_elem(const void *p, int64_t i) {
    if constexpr (sizeof(T) == 2) return bf16_to_f32(from_global<uint16_t>(static_cast<const uint16_t *>(p) + i));
    else return from_global<float>(static_cast<const float *>(p) + i);
}
// Four elements from a multiple of four, as they are stored; widened only when they are used,
// since a load that is widened at once is waited for at once.
template <typename T>
struct Stored;
template <>
struct Stored<float> {
    using four = Float4;
    static __device__ __forceinline__ Float4 widen(Float4 v) { return v; }
    static __device__ __forceinline__ float widen(float v) { return v; }
};
template <>
struct Stored<uint16_t> {
    using four = Uint2;
    static __device__ __forceinline__ Float4 widen(Uint2 v) {
        return {__builtin_bit_cast(float, v.x << 16), __builtin_bit_cast(float, v.x & 0xffff0000u),
                __builtin_bit_cast(float, v.y << 16), __builtin_bit_cast(float, v.y & 0xffff0000u)};
    }
    static __device__ __forceinline__ float widen(uint16_t v) { return bf16_to_f32(v); }
};
template <typename T>
__device__ __forceinline__ typename Stored<T>::four load_four(const void *p, int64_t i) {
    return from_global<typename Stored<T>::four>(static_cast<const T *>(p) + i);
}

// M from the gradient and the updated momentum.
__device__ __forceinline__ float combine(const Hyper &h, float g, float m) {
    return !h.step ? g : h.nesterov ? __builtin_fmaf(h.mu, m, h.rest * g) : m;
}
template <typename T>
__device__ __forceinline__ float source(const Matrix &m, const Hyper &h, int64_t i) {
    const float g = load_elem<T>(m.grad, i);
    return h.step ? combine(h, g, load_elem<float>(m.momentum, i)) : g;
}

// Whether groups of four along a row can be loaded at once.
template <typename T>
__device__ __forceinline__ bool by_four(const Matrix &m, bool step) {
    const uintptr_t p = (uintptr_t)m.grad | (uintptr_t)m.param, q = step ? (uintptr_t)m.momentum : 0;
    return m.cols % 4 == 0 && p % (4 * sizeof(T)) == 0 && q % 16 == 0;
}

// ------------------------------------------------------------------ the table
// The matrices travel as kernel arguments, so a step needs no copy from the host and can be
// captured.
constexpr int kTableChunk = 48;

struct TableChunk {
    Matrix m[kTableChunk];
};

__global__ __launch_bounds__(64) void muon_table(Matrix *dst, TableChunk chunk, int count) {
    if ((int)threadIdx.x < count) dst[threadIdx.x] = chunk.m[threadIdx.x];
}

// D[4 i + l / 16][l % 16] for i = 0..3 of A[l % 16][l / 16] B[l / 16][l % 16].
__device__ __forceinline__ f64x4 mfma_f64(double a, double b, f64x4 c) {
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}

// ------------------------------------------------------------------ Gram matrix, one pass
// A workgroup of 8 waves reads its range of the long side once, with every row of the short
// side, updates the momentum there, and holds the lower triangle of its partial Gram matrix
// in registers, in blocks of 64 x 64: a wave has one block below the diagonal (16 tiles of 16 x
// 16 from 8 operand reads) or two on it (2 x 10 tiles). With 256 rows that makes 6 + 2 waves,
// 36 tiles on the fullest SIMD of 34 on average; with fewer rows groups of 2 waves or single
// waves share out the k-steps and add their sums in LDS at the end. M goes to LDS as doubles: converting
// at the operand reads does it four times over, in the pipe that the products need. Reading M once costs 12 bytes an
// element (4 in orthogonalize); the products, 64 cycles for 16 x 16 x 4, bound it from rank 256 on.
constexpr int kGramThreads = 512;
constexpr int kGramLds = 2 * kChunk * (kOnePass + 16);   // doubles: two stages, 139 KB

template <typename T>
struct Four {
    typename Stored<T>::four g;
    Float4 m;
    __device__ __forceinline__ void set(int e, const T *p) {
        if constexpr (sizeof(T) == 2) g[e / 2] |= (uint32_t)from_global<uint16_t>(p) << 16 * (e % 2);
        else g[e] = from_global<float>(p);
    }
};

template <typename T, int NT, bool TALL>
__device__ __forceinline__ void gram_one_pass(const Matrix &m, const Item &it, const Hyper &h, double *ws, double *lds) {
    constexpr int kRows = 16 * NT, kUnits = kRows * kChunk / 4;
    constexpr int kPasses = (kUnits + kGramThreads - 1) / kGramThreads;
    constexpr int kPitch = TALL ? kRows + 16 : kChunk + 2;
    constexpr int kStage = TALL ? kPitch * kChunk : kPitch * kRows;
    constexpr int kWaves = NT == 16 ? 8 : NT == 8 ? 2 : 1, kGroups = 8 / kWaves, kMost = 20;
    const int r = short_side(m), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int w = wave % kWaves, group = wave / kWaves;
    // Blocks (bi, bj) below the diagonal: (1, 0), (2, 0), (2, 1), (3, 0), ...; or bi = bj and bi + 1.
    constexpr int kBelow = NT == 16 ? 6 : NT == 8 ? 1 : 0;
    const bool below = w < kBelow;
    const int bi = below ? (w < 1 ? 1 : w < 3 ? 2 : 3) : 2 * (w - kBelow);
    const int bj = below ? w - bi * (bi - 1) / 2 : bi;
    const bool four = by_four<T>(m, h.step);
    const int64_t cols = m.cols;
    f64x4 acc[kMost] = {};
    Four<T> held[kPasses];

    // A unit is four elements along a stored row; a thread's units are `gap` rows apart.
    constexpr int kRowUnits = TALL ? kRows / 4 : kChunk / 4, kGap = kGramThreads / kRowUnits;
    const bool active = kUnits >= kGramThreads || tid < kUnits;
    const int along = tid % kRowUnits * 4, across = tid / kRowUnits;
    const int64_t gap = kGap * (TALL ? (int64_t)r : cols);
    int64_t at0 = TALL ? (int64_t)(it.lo + across) * r + along : (int64_t)across * cols + it.lo + along;
    const int64_t next_chunk = TALL ? (int64_t)kChunk * r : kChunk;
    // elements of unit p inside the matrix and the range, in the chunk at k0
    auto left_of = [&](int p, int k0) -> int {
        const int row = across + p * kGap;
        return TALL ? (k0 + row < it.hi ? r - along : 0) : (row < r ? it.hi - k0 - along : 0);
    };
    auto load = [&](int k0) {
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            held[p] = {};
            if (!active) continue;
            const int64_t at = at0 + p * gap;
            const int left = left_of(p, k0);
            if (four && left >= 4) {
                held[p].g = load_four<T>(m.grad, at);
                if (h.step) held[p].m = load_four<float>(m.momentum, at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < left) {
                        held[p].set(e, static_cast<const T *>(m.grad) + at + e);
                        if (h.step) held[p].m[e] = load_elem<float>(m.momentum, at + e);
                    }
            }
        }
    };
    auto store = [&](int k0, double *stage) {
#pragma unroll
        for (int p = 0; p < kPasses; ++p) {
            if (!active) continue;
            Float4 g = Stored<T>::widen(held[p].g), v = held[p].m;
            if (h.step) {
                const int64_t at = at0 + p * gap;
                const int left = left_of(p, k0);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(h.mu, v[e], h.rest * g[e]);
                if (four && left >= 4) {
                    to_global<Float4>(m.momentum + at, v);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (e < left) to_global<float>(m.momentum + at + e, v[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) g[e] = combine(h, g[e], v[e]);
            }
            const int row = across + p * kGap;
            double2 *dst = reinterpret_cast<double2 *>(stage + row * kPitch + along);
            dst[0] = make_double2(g[0], g[1]);
            dst[1] = make_double2(g[2], g[3]);
        }
        at0 += next_chunk;
    };

    int buf = 0;
    if (it.lo < it.hi) {
        load(it.lo);
        store(it.lo, lds);
    }
    __syncthreads();
    for (int k0 = it.lo; k0 < it.hi; k0 += kChunk) {
        const bool more = k0 + kChunk < it.hi;
        if (more) load(k0 + kChunk);
        const double *stage = lds + buf * kStage + (TALL ? (lane >> 4) * kPitch + (lane & 15)
                                                         : (lane & 15) * kPitch + (lane >> 4));
        // operands x of the first block's rows and y of the second's (or of the next diagonal block)
        const double *xs = stage + 4 * bi * (TALL ? 16 : 16 * kPitch);
        const double *ys = stage + 4 * (below ? bj : bi + 1) * (TALL ? 16 : 16 * kPitch);
        constexpr bool kSecond = NT > 4;
#pragma unroll 1
        for (int step = group; step < kChunk / 4; step += kGroups) {
            double x[4], y[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int at = t * (TALL ? 16 : 16 * kPitch) + step * (TALL ? 4 * kPitch : 4);
                if (t < NT) x[t] = xs[at];
                if constexpr (kSecond) y[t] = ys[at];
            }
            if (below) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (64 * bi + 16 * i < r)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[4 * i + j] = mfma_f64(x[i], y[j], acc[4 * i + j]);
            } else {
#pragma unroll
                for (int i = 0; i < (NT < 4 ? NT : 4); ++i)
                    if (64 * bi + 16 * i < r)
#pragma unroll
                        for (int j = 0; j <= i; ++j)
                            acc[i * (i + 1) / 2 + j] = mfma_f64(x[i], x[j], acc[i * (i + 1) / 2 + j]);
                if constexpr (kSecond) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (64 * (bi + 1) + 16 * i < r)
#pragma unroll
                            for (int j = 0; j <= i; ++j)
                                acc[10 + i * (i + 1) / 2 + j] = mfma_f64(y[i], y[j], acc[10 + i * (i + 1) / 2 + j]);
                }
            }
        }
        if (more) store(k0 + kChunk, lds + (buf ^ 1) * kStage);
        __syncthreads();
        buf ^= 1;
    }

    // the squared norm is the trace
    double norm = 0.0;
    if (!below) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * e + (lane >> 4) == (lane & 15)) {
                    norm += acc[i * (i + 1) / 2 + i][e];
                    if constexpr (NT > 4) norm += acc[10 + i * (i + 1) / 2 + i][e];
                }
    }
    double *sums = lds;
    sums[tid] = norm;
    __syncthreads();
    for (int n = kGramThreads / 2; n; n >>= 1) {
        if (tid < n) sums[tid] += sums[tid + n];
        __syncthreads();
    }
    double *part = part_of(m, ws, it.slot);
    if (tid == 0) part[0] = sums[0];
    __syncthreads();
    // the groups' sums, one group after the other, in LDS
    constexpr int kTiles = NT == 1 ? 1 : NT == 2 ? 3 : NT == 4 ? 10 : kMost;
    static_assert(kGroups == 1 || (16 * kBelow + kTiles) * 256 <= kGramLds, "LDS");
    static_assert(2 * kStage <= kGramLds && kGramThreads <= kGramLds, "LDS");
    double *shared = sums + (below ? 16 * w : 16 * kBelow) * 256 + lane;
    if constexpr (kGroups > 1) {
#pragma unroll 1
        for (int g = 0; g < kGroups; ++g) {
            if (group == g) {
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
                    if (t < 16 || !below)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            double *dst = shared + t * 256 + e * 64;
                            *dst = g ? *dst + acc[t][e] : acc[t][e];
                        }
            }
            __syncthreads();
        }
        if (group) return;
    }
    double *tiles = part + part_head(r) + (lane >> 4) * 16 + (lane & 15);
    const int have = tiles16(r);
    auto write = [&](int i, int j, int t) {
        if (i >= have) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) tiles[tile_of(i, j) + 64 * e] = kGroups > 1 ? shared[t * 256 + e * 64] : acc[t][e];
    };
    if (below) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) write(4 * bi + i, 4 * bj + j, 4 * i + j);
    } else {
#pragma unroll
        for (int i = 0; i < (NT < 4 ? NT : 4); ++i)
#pragma unroll
            for (int j = 0; j <= i; ++j) {
                write(4 * bi + i, 4 * bi + j, i * (i + 1) / 2 + j);
                if constexpr (NT > 4) write(4 * bi + 4 + i, 4 * bi + 4 + j, 10 + i * (i + 1) / 2 + j);
            }
    }
}

// NT for a short side: tiles of 16 rows, rounded up to a power of two.
__host__ __device__ __forceinline__ int one_pass_tiles(int r) {
    return r <= 16 ? 1 : r <= 32 ? 2 : r <= 64 ? 4 : r <= 128 ? 8 : 16;
}

template <typename T, bool TALL>
__device__ __forceinline__ void gram_by_size(const Matrix &m, const Item &it, const Hyper &h, double *ws, double *lds) {
    switch (one_pass_tiles(short_side(m))) {
        case 1: return gram_one_pass<T, 1, TALL>(m, it, h, ws, lds);
        case 2: return gram_one_pass<T, 2, TALL>(m, it, h, ws, lds);
        case 4: return gram_one_pass<T, 4, TALL>(m, it, h, ws, lds);
        case 8: return gram_one_pass<T, 8, TALL>(m, it, h, ws, lds);
        default: return gram_one_pass<T, 16, TALL>(m, it, h, ws, lds);
    }
}

template <typename T>
__global__ __launch_bounds__(kGramThreads, 2) void muon_gram(const Matrix *matrices, const Item *items, Hyper h,
                                                            double *ws) {
    __shared__ __align__(16) double lds[kGramLds];
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    if (m.rows > m.cols) gram_by_size<T, true>(m, it, h, ws, lds);
    else gram_by_size<T, false>(m, it, h, ws, lds);
}

// ------------------------------------------------------------------ Gram matrix, any short side
template <typename T>
__global__ __launch_bounds__(kThreads) void muon_momentum(const Matrix *matrices, const Item *items, Hyper h) {
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    const int r = short_side(m);
    for (int64_t i = (int64_t)it.lo * r + threadIdx.x; i < (int64_t)it.hi * r; i += kThreads)
        to_global<float>(m.momentum + i, __builtin_fmaf(h.mu, load_elem<float>(m.momentum, i), h.rest * load_elem<T>(m.grad, i)));
}

// One 64 x 64 tile (i >= j) of M M^T over the columns lo .. hi - 1: 4 waves of 32 x 32.
template <typename T>
__global__ __launch_bounds__(kThreads) void muon_gram_tiles(const Matrix *matrices, const Item *items, Hyper h,
                                                           double *ws) {
    constexpr int KC = 16, kPitch = KC + 4;
    __shared__ float sa[kGramTile * kPitch], sb[kGramTile * kPitch];
    __shared__ double diagonal[kGramTile];
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    const int r = short_side(m), lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const bool tall = m.rows > m.cols;
    const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
    f64x4 acc[2][2] = {};
    for (int k0 = it.lo; k0 < it.hi; k0 += KC) {
        __syncthreads();
        for (int e = threadIdx.x; e < kGramTile * KC; e += kThreads) {
            const int row = tall ? e % kGramTile : e / KC, k = tall ? e / kGramTile : e % KC;
            auto at = [&](int short_index) -> float {
                if (short_index >= r || k0 + k >= it.hi) return 0.0f;
                return source<T>(m, h, tall ? (int64_t)(k0 + k) * r + short_index
                                            : (int64_t)short_index * m.cols + k0 + k);
            };
            sa[row * kPitch + k] = at(it.i * kGramTile + row);
            sb[row * kPitch + k] = at(it.j * kGramTile + row);
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < KC; s += 4) {
            double a[2], b[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                a[t] = sa[(wi + 16 * t + (lane & 15)) * kPitch + s + (lane >> 4)];
                b[t] = sb[(wj + 16 * t + (lane & 15)) * kPitch + s + (lane >> 4)];
            }
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) acc[x][y] = mfma_f64(a[x], b[y], acc[x][y]);
        }
    }
    double *part = part_of(m, ws, it.slot), *tiles = part + part_head(r);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            const int i = it.i * 4 + wi / 16 + x, j = it.j * 4 + wj / 16 + y;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 4 * e + (lane >> 4), col = lane & 15;
                if (i >= j && i < tiles16(r)) tiles[tile_of(i, j) + row * 16 + col] = acc[x][y][e];
                if (i == j && row == col) diagonal[wi + 16 * x + row] = acc[x][y][e];
            }
        }
    if (it.i != it.j) return;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
        for (int e = 0; e < kGramTile; ++e) sum += diagonal[e];
        part[it.i] = sum;
    }
}

// 1 / max(|M|, eps) from the parts' squared norms: every wave for itself, in one fixed order.
__device__ __forceinline__ double inverse_norm(const Matrix &m, double *ws, double eps) {
    const int r = short_side(m), heads = r <= kOnePass ? 1 : (r + kGramTile - 1) / kGramTile;
    double sum = 0.0;
    for (int i = threadIdx.x & 63; i < m.splits * heads; i += 64) sum += part_of(m, ws, i / heads)[i % heads];
#pragma unroll
    for (int n = 32; n; n >>= 1) sum += __shfl_xor(sum, n, 64);
    const double norm = sqrt(sum);
    return 1.0 / (norm < eps ? eps : norm);
}

// Element `e` of tile (i, j): the parts in order.
__device__ __forceinline__ double join_tile(const Matrix &m, double *ws, int i, int j, int e) {
    const double *p = part_of(m, ws, 0) + part_head(short_side(m)) + tile_of(i, j) + e;
    const int64_t step = part_size(short_side(m));
    double v = 0.0;
#pragma unroll 8
    for (int s = 0; s < m.splits; ++s) v += p[s * step];
    return v;
}

// One 16 x 16 tile of G.
__global__ __launch_bounds__(kThreads) void muon_join(const Matrix *matrices, const Item *items, Hyper h, double *ws) {
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    const int rp = padded(short_side(m)), row = threadIdx.x >> 4, col = threadIdx.x & 15;
    const double inv = inverse_norm(m, ws, h.eps);
    if (it.i == 0 && threadIdx.x == 0) ws[m.scratch] = inv;
    double *g = buffer(m, ws, kG);
    const int64_t i = it.i * 16 + row, j = it.j * 16 + col;
    if (it.i >= tiles16(short_side(m))) {   // padding rows
        g[i * rp + j] = g[j * rp + i] = 0.0;
        return;
    }
    double v = join_tile(m, ws, it.i, it.j, threadIdx.x) * (inv * inv);
    if (i == j && i < short_side(m)) v += gram_floor(short_side(m));
    if (i >= j) g[i * rp + j] = g[j * rp + i] = v;
}

// ------------------------------------------------------------------ short sides up to 64
// All steps in one workgroup of 8 waves, G, P, T and Q in LDS. Symmetric operands are read
// along rows for both sides of a product (16 columns of 4 rows a load: odd rows are stored with
// their blocks of 16 columns exchanged in pairs, so two rows fill the banks); the ten tiles (i
// >= j) of rank 64 go to the waves in turn, all of a tile's loads in flight at once and its
// products in two chains.
constexpr int kSmallThreads = 512;

__global__ __launch_bounds__(kSmallThreads) void muon_small(const Matrix *matrices, const Item *items, Hyper h,
                                                           double *ws, int steps) {
    constexpr int kMost = 10 * 256 / kSmallThreads;
    __shared__ double sg[kSmall * kSmall], sp[kSmall * kSmall], st[kSmall * kSmall], sq[kSmall * kSmall];
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    const int r = short_side(m), n = tiles16(r), count = n * (n + 1) / 2, tid = threadIdx.x, lane = tid & 63,
              wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    auto at = [](int row, int col) { return row * kSmall + (col ^ ((row & 1) << 4)); };
    auto tile_row = [](int t) { return t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3; };
    const double inv = inverse_norm(m, ws, h.eps);
    {
        // the parts in order, all of a thread's elements at once
        const double *p = part_of(m, ws, 0) + part_head(r) + tid;
        const int64_t step = part_size(r);
        double v[kMost] = {};
#pragma unroll 8
        for (int s = 0; s < m.splits; ++s)
#pragma unroll
            for (int x = 0; x < kMost; ++x)
                if (x * kSmallThreads + tid < count * 256) v[x] += p[s * step + x * kSmallThreads];
#pragma unroll
        for (int x = 0; x < kMost; ++x) {
            const int t = (x * kSmallThreads + tid) >> 8, i = tile_row(t), j = t - i * (i + 1) / 2;
            const int row = i * 16 + ((tid & 255) >> 4), col = j * 16 + (tid & 15);
            if (t < count && row >= col)
                sg[at(row, col)] = sg[at(col, row)] = v[x] * (inv * inv) + (row == col && row < r ? gram_floor(r) : 0.0);
        }
    }
    __syncthreads();

    // dst = left right + diagonal I, or a I + b left + c left right; dst may be an operand.
    auto product = [&](const double *left, const double *right, double *dst, bool polynomial, double diagonal = 0.0) {
        f64x4 result[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int t = wave + 8 * x;
            if (t >= count) continue;
            const int i = tile_row(t), j = t - i * (i + 1) / 2;
            const int a = at(lane >> 4, 16 * i + (lane & 15)), b = at(lane >> 4, 16 * j + (lane & 15));
            double p[16], q[16];   // k = 4 u + lane / 16
#pragma unroll
            for (int u = 0; u < 16; ++u)
                if (u < 4 * n) {
                    p[u] = left[a + 4 * u * kSmall];
                    q[u] = right[b + 4 * u * kSmall];
                }
            f64x4 even = {}, odd = {};
#pragma unroll
            for (int u = 0; u < 16; u += 2)
                if (u < 4 * n) {
                    even = mfma_f64(p[u], q[u], even);
                    odd = mfma_f64(p[u + 1], q[u + 1], odd);
                }
            result[x] = even + odd;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * i + 4 * e + (lane >> 4), col = 16 * j + (lane & 15);
                if (polynomial) result[x][e] = h.c * result[x][e] + h.b * left[at(row, col)];
                if (row == col && row < r) result[x][e] += polynomial ? h.a : diagonal;
            }
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int t = wave + 8 * x;
            if (t >= count) continue;
            const int i = tile_row(t), j = t - i * (i + 1) / 2;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = 16 * i + 4 * e + (lane >> 4), col = 16 * j + (lane & 15);
                if (row >= col) dst[at(row, col)] = dst[at(col, row)] = result[x][e];
            }
        }
        __syncthreads();
    };
    for (int i = 0; i < steps; ++i) {
        double *p = i == 0 ? sq : sp;   // the first P is the first Q
        product(sg, sg, p, true);
        if (i + 1 < steps) product(p, sg, st, false);
        if (i) product(p, sq, sq, false);
        if (i + 1 < steps) product(p, st, sg, false, gram_floor(r));
    }
    const int rp = padded(r);
    float *final = final_q(m, ws);
    for (int e = tid; e < rp * rp; e += kSmallThreads) {
        const int row = e % rp, k = e / rp;
        final[final_at(rp, row, k)] = row < 16 * n && k < 16 * n ? (float)(sq[at(row, k)] * inv) : 0.0f;
    }
}

// ------------------------------------------------------------------ r x r products
enum StageKind { kMakeP = 0, kMultiply = 1 };

struct StageOp {
    int kind, left, right, dst, last;
};

// One 32 x 32 tile (i >= j) of left right, both symmetric and commuting, so their product is
// symmetric too and the tile's mirror image is its transpose. kMakeP: a I + b G + c G G. Each
// of the 8 waves takes an eighth of the reduction over the whole tile (one load per product
// instead of two) straight from L2, all loads of up to kSteps k-steps in flight at once, operand
// rows read along k's rows (symmetry), and the sums are added in LDS in order.
constexpr int kStageThreads = 512;

__global__ __launch_bounds__(kStageThreads) void muon_stage(const Matrix *matrices, const Item *items, Hyper h,
                                                           double *ws, StageOp op0, StageOp op1) {
    constexpr int kPitch = kPad + 1, kSteps = 4;
    __shared__ double sums[4][kPad * kPitch];
    const StageOp op = blockIdx.y ? op1 : op0;
    const Item it = items[blockIdx.x];
    if (it.matrix < 0) return;
    const Matrix m = matrices[it.matrix];
    const int r = short_side(m), rp = padded(r), lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);   // scalar, as all that follows from it
    const int64_t lane_at = (lane & 15) + (int64_t)(lane >> 4) * rp;
    const double *left = buffer(m, ws, op.left) + it.i * kPad + lane_at;
    const double *right = buffer(m, ws, op.right) + it.j * kPad + lane_at;
    f64x4 acc[2][2] = {};
    const int steps = rp / 32, first = wave * steps;   // k-steps of 4 rows
    for (int s0 = 0; s0 < steps; s0 += kSteps) {
        double x[kSteps][2], y[kSteps][2];
#pragma unroll
        for (int u = 0; u < kSteps; ++u)
            if (s0 + u < steps) {
                const int64_t at = (int64_t)(first + s0 + u) * 4 * rp;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    x[u][t] = left[at + 16 * t];
                    y[u][t] = right[at + 16 * t];
                }
            }
#pragma unroll
        for (int u = 0; u < kSteps; ++u)
            if (s0 + u < steps)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = mfma_f64(x[u][i], y[u][j], acc[i][j]);
    }
    // waves 4 - 7, then 0 - 3 on top of them
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        if (wave >> 2 != pass) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        double *dst = &sums[wave & 3][(16 * i + 4 * e + (lane >> 4)) * kPitch + 16 * j + (lane & 15)];
                        *dst = pass ? *dst + acc[i][j][e] : acc[i][j][e];
                    }
        }
        __syncthreads();
    }
    const double inv = op.last ? ws[m.scratch] : 1.0;
    const double *g = buffer(m, ws, op.left);
    double *dst = buffer(m, ws, op.dst);
    float *final = final_q(m, ws);
    auto value = [&](int row, int col) -> double {
        const int at = row * kPitch + col;
        double v = ((sums[0][at] + sums[1][at]) + sums[2][at]) + sums[3][at];
        if (op.kind == kMakeP) {
            const int i = it.i * kPad + row, j = it.j * kPad + col;
            v = h.c * v + h.b * g[(int64_t)i * rp + j];
            if (i == j && i < r) v += h.a;
        } else if (op.dst == kG && it.i == it.j && row == col && it.i * kPad + row < r) {
            v += gram_floor(r);
        }
        return v;
    };
    for (int e = threadIdx.x; e < kPad * kPad; e += kStageThreads) {
        const int row = e / kPad, col = e % kPad;
        // (row, col) of the tile itself, then of its mirror image, both stored along rows
        const double v = it.i == it.j && row < col ? value(col, row) : value(row, col);
        const int i = it.i * kPad + row, j = it.j * kPad + col;
        if (op.last) final[final_at(rp, i, j)] = (float)(v * inv);
        else dst[(int64_t)i * rp + j] = v;
        if (it.i != it.j) {
            const double u = value(col, row);
            const int x = it.j * kPad + row, y = it.i * kPad + col;
            if (op.last) final[final_at(rp, x, y)] = (float)(u * inv);
            else dst[(int64_t)x * rp + y] = u;
        }
    }
}

// ------------------------------------------------------------------ the last product
// Q M by 8 waves: each takes 32 rows of the short side and 64 elements of the long side
// (v_mfma_f32_32x32x2, 2 x 32), so a slab covers 64, 128, 256 or 512 elements of the long side
// with short sides up to 256, 128, 64 or 32. Its part of M (combined from gradient and momentum
// on the way) lies in LDS, Q comes from L2 in the order that final_at gives it.
// One workgroup per CU runs through an even share of all slabs, of several matrices if it has
// to. Loads return in the order they were asked for, so a slab's product is cut into groups of
// 32 of the reduction, and each group asks first for the next group's Q, then for a part of
// the next slab's gradient and momentum and of its own parameters: those have a group's
// products (1.7 us) to come in before anything waits behind them. Two layers' adapters of rank
// 256 took 240 us (five passes, a cold card); a slab per workgroup, two workgroups per CU with
// nothing asked for ahead, 302. Short sides past 256 go slab by slab, in blocks of 256 rows and 256 of the reduction.
constexpr int kApplyThreads = 512;
constexpr int kApplyLds = 18432;   // floats: 256 x 72, 128 x 136, 64 x 264, 32 x 520 and their transposes

__host__ __device__ __forceinline__ int apply_blocks(int r) { return r <= 32 ? 1 : r <= 64 ? 2 : r <= 128 ? 4 : 8; }

// acc[t] += Q[32 rows, 32] M[32, 2 x 32 elements of the long side]; q: what the lane has of Q.
template <int PITCH, bool TALL>
__device__ __forceinline__ void apply_product(f32x16 (&acc)[2], const float4 (&q)[4], const float *sx, int part, int lane) {
    const int half = lane >> 5;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int s = 8 * i + 4 * half;
        const float qv[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int l = part + 32 * t + (lane & 31);
            float xv[4];
            if constexpr (TALL) {
                const float4 x4 = *reinterpret_cast<const float4 *>(sx + l * PITCH + s);
                xv[0] = x4.x; xv[1] = x4.y; xv[2] = x4.z; xv[3] = x4.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) xv[e] = sx[(s + e) * PITCH + l];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                acc[t] = TALL ? __builtin_amdgcn_mfma_f32_32x32x2f32(xv[e], qv[e], acc[t], 0, 0, 0)
                              : __builtin_amdgcn_mfma_f32_32x32x2f32(qv[e], xv[e], acc[t], 0, 0, 0);
        }
    }
}

// Where a lane's results go: register i is `8 (i / 4) + i % 4` rows of the stored matrix below
// the lane's first, of which `limit` exist; a parameter that does not exist reads another.
template <typename T, bool TALL>
struct ApplyPlace {
    T *param;
    int64_t stride;
    int limit;
    __device__ __forceinline__ ApplyPlace(const Matrix &m, int r, int64_t width, int row, int64_t col, int lane) {
        const int half = lane >> 5, s = row + (TALL ? lane & 31 : 4 * half);
        const int64_t l = col + (TALL ? 4 * half : lane & 31);
        stride = TALL ? r : m.cols;
        const int64_t below = TALL ? (s < r ? width - l : 0) : (l < width ? r - s : 0);
        limit = below > 32 ? 32 : below < 0 ? 0 : (int)below;
        param = static_cast<T *>(m.param) + (limit ? (TALL ? l * r + s : (int64_t)s * m.cols + l) : 0);
    }
    __device__ static __forceinline__ int down(int i) { return 8 * (i >> 2) + (i & 3); }
    __device__ __forceinline__ T load(int i) const {
        const int last = limit > 1 ? limit - 1 : 0;
        return from_global<T>(param + (uint64_t)(uint32_t)(down(i) < last ? down(i) : last) * (uint32_t)stride);
    }
    // acc = old keep - lr adjust acc
    __device__ static __forceinline__ void update(f32x16 &acc, const T (&old)[16], const Hyper &h, const Matrix &m) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            acc[i] = __builtin_fmaf(-h.lr * m.adjust, acc[i], Stored<T>::widen(old[i]) * h.keep);
    }
    __device__ __forceinline__ void store(const f32x16 &v) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (down(i) >= limit) continue;
            if constexpr (sizeof(T) == 2) to_global<uint16_t>(param + down(i) * stride, bf16_bits(v[i]));
            else to_global<float>(param + down(i) * stride, v[i]);
        }
    }
};

template <typename T, int NB, bool TALL, bool STEP>
__device__ __forceinline__ void apply_run(const Matrix &m, const Item &it, const Hyper &h, double *ws, float *lds) {
    constexpr int kLong = 64 * (8 / NB), kShort = 32 * NB;
    constexpr int kPitch = TALL ? kShort + 4 : kLong + 8;
    constexpr int kUnits = kLong * kShort / 4 / kApplyThreads;   // 8, of four elements along a stored row
    constexpr int kRowUnits = TALL ? kShort / 4 : kLong / 4, kGap = kApplyThreads / kRowUnits;
    static_assert(kPitch * (TALL ? kLong : kShort) <= kApplyLds && kUnits == 8, "LDS");
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));   // keeps the variants' addresses apart: shared ones spill
    const int r = short_side(m), rp = padded(r), lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row = 32 * (wave % NB), part = wave / NB * 64;
    const int64_t width = TALL ? m.rows : m.cols;
    const bool four = by_four<T>(m, STEP);
    const int along = tid % kRowUnits * 4, across = tid / kRowUnits;
    Four<T> held[kUnits];
    // Past the matrix's end its last elements come instead: Q has zeros for the short side's
    // (whose groups past rp are left out), the long side's results are not stored.
    auto fetch = [&](int p, int64_t col0) {
        const int line = across + p * kGap;
        const int64_t left = width - col0;
        const int down = TALL ? (int)least(line, left - 1) : least(line, r - 1);
        const int right = TALL ? (int)least(along, r - 4) : (int)least(along, left - 4);
        const int64_t at = (uint64_t)(uint32_t)down * (uint32_t)m.cols + (TALL ? col0 * m.cols : col0) + right;
        held[p].g = load_four<T>(m.grad, at);
        if constexpr (STEP) held[p].m = load_four<float>(m.momentum, at);
    };
    // Q of this wave's rows, group by group; a wave past the last row reads the last ones'.
    const float4 *q = reinterpret_cast<const float4 *>(final_q(m, ws)) + (row < rp ? row : rp - 32) * 2;
    unsigned q_lane = (lane & 31) * 2 + half;
    int q_step = rp * 2;
    auto q_at = [&](int group, int i) { return (q + (4 * group + i) * q_step)[q_lane]; };
    float4 now[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) now[i] = q_at(0, i);
    auto keep = [&](int p, float *sx) {
        Float4 x = Stored<T>::widen(held[p].g);
        if constexpr (STEP)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = combine(h, x[e], held[p].m[e]);
        *reinterpret_cast<Float4 *>(sx + (across + p * kGap) * kPitch + along) = x;
    };
    if (four) {
#pragma unroll
        for (int p = 0; p < kUnits; ++p) fetch(p, it.lo);
#pragma unroll
        for (int p = 0; p < kUnits; ++p) keep(p, lds);
    }
    float *sx = lds, *other = lds + kApplyLds;
    for (int64_t col0 = it.lo; col0 < it.hi; col0 += kLong) {
        if (!four) {
#pragma unroll 4
            for (int u = tid; u < kLong * kShort; u += kApplyThreads) {
                const int s = TALL ? u % kShort : u / kLong, l = TALL ? u / kShort : u % kLong;
                const int64_t at = TALL ? (col0 + l) * r + s : s * m.cols + col0 + l;
                sx[TALL ? l * kPitch + s : s * kPitch + l] = s < r && col0 + l < width ? source<T>(m, h, at) : 0.0f;
            }
        }
        __syncthreads();
        const bool more = four && col0 + kLong < it.hi;
        const ApplyPlace<T, TALL> first(m, r, width, row, col0 + part, lane);
        const ApplyPlace<T, TALL> second(m, r, width, row, col0 + part + 32, lane);
        T old[2][16];
        f32x16 acc[2] = {};
#pragma unroll
        for (int group = 0; group < NB; ++group) {
            float4 ahead[4];
            const int next = 32 * (group + 1) < rp ? group + 1 : 0;
            asm volatile("" : "+v"(q_lane), "+s"(q_step));   // nor are the addresses kept from slab to slab
#pragma unroll
            for (int i = 0; i < 4; ++i) ahead[i] = q_at(next, i);
#pragma unroll
            for (int p = 0; p < kUnits; ++p) {   // over the first three quarters of the groups
                if (p * 3 * NB / 32 != group) continue;
                if (more) fetch(p, col0 + kLong);
                if constexpr (STEP)
#pragma unroll
                    for (int i = 2 * p; i < 2 * p + 2; ++i) {
                        old[0][i] = first.load(i);
                        old[1][i] = second.load(i);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (row < rp && 32 * group < rp)
                apply_product<kPitch, TALL>(acc, now, sx + 32 * group * (TALL ? 1 : kPitch), part, lane);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int p = 0; p < kUnits; ++p)   // what has had a group's time or two
                if (group == least(NB - 1, p * 3 * NB / 32 + NB / 4) && more) keep(p, other);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) now[i] = ahead[i];
        }
        if constexpr (STEP) {
            first.update(acc[0], old[0], h, m);
            second.update(acc[1], old[1], h, m);
        }
        first.store(acc[0]);
        second.store(acc[1]);
        float *swap = sx;
        sx = other;
        other = swap;
    }
}

// Slabs of a matrix whose short side is past 256.
template <typename T, bool TALL, bool STEP>
__device__ __forceinline__ void apply_blocked(const Matrix &m, const Item &it, const Hyper &h, double *ws, float *sx) {
    constexpr int kLong = 64, kShort = 256, kPitch = TALL ? kShort + 4 : kLong + 8;
    const int r = short_side(m), rp = padded(r), tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t width = TALL ? m.rows : m.cols;
    const int blocks = (rp + kShort - 1) / kShort;
    for (int64_t n = 0; n < (it.hi - it.lo + kLong - 1) / kLong * blocks; ++n) {
        const int64_t col0 = it.lo + n / blocks * kLong;
        const int row = (int)(n % blocks) * kShort + 32 * wave;
        f32x16 acc[2] = {};
        for (int k0 = 0; k0 < rp; k0 += kShort) {
            __syncthreads();
#pragma unroll 4
            for (int u = tid; u < kLong * kShort; u += kApplyThreads) {
                const int s = TALL ? u % kShort : u / kLong, l = TALL ? u / kShort : u % kLong;
                const bool inside = k0 + s < r && col0 + l < width;
                const int64_t at = TALL ? (col0 + l) * r + k0 + s : (k0 + s) * m.cols + col0 + l;
                sx[TALL ? l * kPitch + s : s * kPitch + l] = inside ? source<T>(m, h, at) : 0.0f;
            }
            __syncthreads();
            if (row >= rp) continue;
            const float4 *q = reinterpret_cast<const float4 *>(final_q(m, ws)) + (row + (lane & 31)) * 2 + (lane >> 5);
            for (int s = 0; s < kShort && k0 + s < rp; s += 32) {
                float4 now[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) now[i] = q[((int64_t)(k0 + s) / 8 + i) * rp * 2];
                apply_product<kPitch, TALL>(acc, now, sx + s * (TALL ? 1 : kPitch), 0, lane);
            }
        }
        if (row >= rp) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const ApplyPlace<T, TALL> place(m, r, width, row, col0 + 32 * t, lane);
            if constexpr (STEP) {
                T old[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) old[i] = place.load(i);
                place.update(acc[t], old, h, m);
            }
            place.store(acc[t]);
        }
    }
}

template <typename T, bool TALL, bool STEP>
__device__ __forceinline__ void apply_by_size(const Matrix &m, const Item &it, const Hyper &h, double *ws, float *lds) {
    if (short_side(m) > 256) return apply_blocked<T, TALL, STEP>(m, it, h, ws, lds);
    switch (apply_blocks(short_side(m))) {
        case 1: return apply_run<T, 1, TALL, STEP>(m, it, h, ws, lds);
        case 2: return apply_run<T, 2, TALL, STEP>(m, it, h, ws, lds);
        case 4: return apply_run<T, 4, TALL, STEP>(m, it, h, ws, lds);
        default: return apply_run<T, 8, TALL, STEP>(m, it, h, ws, lds);
    }
}

// An item's slot names the item that the same workgroup takes next, if any; those have pad0 = 1.
template <typename T, bool STEP>
__global__ __launch_bounds__(kApplyThreads, 2) void muon_apply(const Matrix *matrices, const Item *items, Hyper h,
                                                              double *ws) {
    __shared__ __align__(16) float lds[2 * kApplyLds];
    Item it = items[blockIdx.x];
    if (it.pad0) return;
    for (;;) {
        const Matrix m = matrices[it.matrix];
        if (m.rows > m.cols) apply_by_size<T, true, STEP>(m, it, h, ws, lds);
        else apply_by_size<T, false, STEP>(m, it, h, ws, lds);
        if (!it.slot) break;
        it = items[it.slot];
        __syncthreads();
    }
}

// ------------------------------------------------------------------ host side
constexpr int64_t kMaxShort = 16384, kMaxLong = (int64_t)1 << 30;
constexpr int64_t kGroupsWanted = 256;   // one Gram workgroup per CU

enum { kItemsGram = 0, kItemsTiles, kItemsMomentum, kItemsJoin, kItemsStage, kItemsSmall, kItemsApply, kKinds };

struct Shape {
    int r, rp;
    int64_t width;
};

bool shape_of(int64_t rows, int64_t cols, Shape &s) {
    if (rows <= 0 || cols <= 0) return false;
    s.width = std::max(rows, cols);
    if (std::min(rows, cols) > kMaxShort || s.width > kMaxLong) return false;
    s.r = (int)std::min(rows, cols);
    s.rp = padded(s.r);
    return true;
}

// Workgroups go to the 8 XCDs in turn: hands each XCD one run of neighbouring items, so that
// what they share stays in its L2. Padded with items of no matrix to whole turns.
void by_xcd(std::vector<Item> &items) {
    constexpr int64_t kXcds = 8;
    const int64_t n = (int64_t)items.size(), run = cdiv(n, kXcds);
    std::vector<Item> ordered((size_t)(run * kXcds), Item{-1, 0, 0, 0, 0, 0, 0, 0});
    for (int64_t x = 0, from = 0; x < kXcds; ++x) {
        const int64_t to = n * (x + 1) / kXcds;
        for (int64_t k = 0; from < to; ++k, ++from) ordered[(size_t)(k * kXcds + x)] = items[(size_t)from];
    }
    items.swap(ordered);
}

int64_t scratch_doubles(const Shape &s) {
    const int64_t square = (int64_t)s.rp * s.rp;
    return 2 + (s.r <= kSmall ? 0 : kBuffers * square) + square / 2;
}

int status_of_last_launch() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : (int)e;
}

// Cost of a chunk of the long side in the one-pass Gram kernel, in its unit of time: a tile's
// product on one of four SIMDs, and no less than about 4 for reading the chunk.
int64_t chunk_cost(int r) {
    const int64_t t = one_pass_tiles(r);
    return std::max<int64_t>(4, t * (t + 1) / 2);
}

// Long-side elements per workgroup so that none takes longer than `cap`, in whole chunks; at
// least two, which pays for the partial result, and for short sides up to kSmall, whose one
// workgroup adds all parts, so many that a chunk's time (0.7 us) and a part's (1.1 us) balance:
// 2049 x 64 in 33 parts 10 + 96 us, in 7 17 + 64.
int64_t gram_step(const Shape &s, int64_t cap) {
    int64_t chunks = std::max<int64_t>(2, cap / chunk_cost(s.r));
    if (s.r <= kSmall) chunks = std::max<int64_t>(chunks, (int64_t)sqrt(1.6 * (double)cdiv(s.width, kChunk)));
    return chunks * kChunk;
}

// The smallest cap with which all the one-pass Gram items run at once.
int64_t gram_cap(const std::vector<Shape> &shapes) {
    int64_t low = 1, high = 1;
    auto fits = [&](int64_t cap) {
        int64_t n = 0;
        for (const Shape &s : shapes)
            if (s.r <= kOnePass) n += cdiv(s.width, gram_step(s, cap));
        return n <= std::max<int64_t>(kGroupsWanted, (int64_t)shapes.size());
    };
    while (!fits(high) && high < (int64_t)1 << 40) high *= 2;
    while (low < high) {
        const int64_t mid = (low + high) / 2;
        if (fits(mid)) high = mid;
        else low = mid + 1;
    }
    return high;
}

// The last product's slabs in even shares, one per CU. A slab of a short side past 256 costs
// its blocks' products.
void share_slabs(const std::vector<Shape> &shapes, std::vector<Item> &items) {
    int64_t total = 0, slabs = 0, done = 0, last = -1;
    auto length = [](const Shape &s) -> int64_t { return 64 * (8 / apply_blocks(s.r)); };
    auto cost = [](const Shape &s) { return cdiv(s.r, 256) * cdiv(s.r, 256); };
    for (const Shape &s : shapes) {
        slabs += cdiv(s.width, length(s));
        total += cdiv(s.width, length(s)) * cost(s);
    }
    const int64_t shares = std::min(slabs, kGroupsWanted);
    std::vector<Item> more;
    std::vector<int32_t> owner;   // of each in `more`: the share it belongs to
    for (size_t i = 0; i < shapes.size(); ++i) {
        const Shape &s = shapes[i];
        const int64_t slab = length(s), count = cdiv(s.width, slab);
        for (int64_t c = 0, n; c < count; c += n) {
            const int64_t share = done * shares / total, end = cdiv((share + 1) * total, shares);
            n = std::min(count - c, cdiv(end - done, cost(s)));
            const Item it = {(int32_t)i, 0, 0, (int32_t)(c * slab), (int32_t)std::min(s.width, (c + n) * slab), 0, share == last, 0};
            if (it.pad0) {
                more.push_back(it);
                owner.push_back((int32_t)items.size() - 1);
            } else {
                items.push_back(it);
            }
            last = share;
            done += n * cost(s);
        }
    }
    const int32_t firsts = (int32_t)items.size();
    for (size_t k = 0; k < more.size(); ++k) {
        const int32_t index = firsts + (int32_t)k;
        if (k && owner[k - 1] == owner[k]) items.back().slot = index;
        else items[(size_t)owner[k]].slot = index;
        items.push_back(more[k]);
    }
}

// A matrix's items and its number of partial Gram matrices.
void plan_matrix(int32_t index, const Shape &s, int64_t cap, std::vector<Item> (&items)[kKinds], int32_t &splits) {
    const bool one_pass = s.r <= kOnePass;
    const int64_t blocks = cdiv(s.r, kGramTile) * (cdiv(s.r, kGramTile) + 1) / 2;
    const int64_t parts = one_pass ? cdiv(s.width, gram_step(s, cap))
                                   : std::max<int64_t>(1, std::min<int64_t>(cdiv(s.width, 512), 1024 / blocks));
    const int64_t step = cdiv(cdiv(s.width, parts), kChunk) * kChunk;   // even parts
    const int64_t count = cdiv(s.width, step);
    auto range = [&](int64_t k, int32_t i, int32_t j) -> Item {
        return {index, i, j, (int32_t)(k * step), (int32_t)std::min(s.width, (k + 1) * step), (int32_t)k, 0, 0};
    };
    if (one_pass) {
        for (int64_t k = 0; k < count; ++k) items[kItemsGram].push_back(range(k, 0, 0));
    } else {
        const int tiles = (s.r + kGramTile - 1) / kGramTile;
        for (int64_t k = 0; k < count; ++k)
            for (int a = 0; a < tiles; ++a)
                for (int b = 0; b <= a; ++b) items[kItemsTiles].push_back(range(k, a, b));
        for (int64_t c = 0; c < s.width; c += 64)
            items[kItemsMomentum].push_back({index, 0, 0, (int32_t)c, (int32_t)std::min(s.width, c + 64), 0, 0, 0});
    }
    splits = (int32_t)count;
    if (s.r <= kSmall) {
        items[kItemsSmall].push_back({index, 0, 0, 0, 0, 0, 0, 0});
    } else {
        for (int a = 0; a < s.rp / 16; ++a)
            for (int b = 0; b <= a; ++b) items[kItemsJoin].push_back({index, a, b, 0, 0, 0, 0, 0});
        for (int a = 0; a < s.rp / kPad; ++a)
            for (int b = 0; b <= a; ++b) items[kItemsStage].push_back({index, a, b, 0, 0, 0, 0, 0});
    }
}

}  // namespace
}  // namespace ct

using namespace ct;

static_assert(sizeof(Matrix) == sizeof(ct_muon_matrix) && sizeof(Matrix) % 8 == 0, "ct_muon_matrix");
static_assert(sizeof(TableChunk) < 3600, "kernel arguments");
static_assert(kKinds == CT_MUON_KINDS, "counts");

extern "C" int ct_muon_plan(ct_muon_matrix *matrices, int64_t count, int32_t *entries, int64_t capacity,
                            int64_t *counts, int64_t *workspace_bytes) {
    if (count < 0 || count > 1 << 24) return -CT_EINVAL_SHAPE;
    if (!counts || !workspace_bytes || (count && !matrices)) return -CT_EINVAL_POINTER;
    try {
        std::vector<Item> items[kKinds];
        std::vector<Shape> shapes((size_t)count);
        for (int64_t i = 0; i < count; ++i)
            if (!shape_of(matrices[i].rows, matrices[i].cols, shapes[(size_t)i])) return -CT_EINVAL_SHAPE;
        const int64_t cap = gram_cap(shapes);
        // the table, then each matrix's partials and buffers, all 16-byte aligned
        int64_t doubles = cdiv(count * (int64_t)sizeof(Matrix), 16) * 2;
        for (int64_t i = 0; i < count; ++i) {
            const Shape &s = shapes[(size_t)i];
            plan_matrix((int32_t)i, s, cap, items, matrices[i].splits);
            matrices[i].parts = doubles;
            doubles += matrices[i].splits * part_size(s.r);
            matrices[i].scratch = doubles;
            doubles += scratch_doubles(s);
        }
        share_slabs(shapes, items[kItemsApply]);
        by_xcd(items[kItemsStage]);
        int64_t size = 0;
        for (int k = 0; k < kKinds; ++k) {
            counts[k] = (int64_t)items[k].size();
            if (counts[k] > 0x7fffffff / kGramThreads) return -CT_EINVAL_SHAPE;
            size += counts[k];
        }
        *workspace_bytes = doubles * (int64_t)sizeof(double);
        if (!entries) return 0;
        if (capacity < size) return -CT_EINVAL_WORKSPACE;
        Item *dst = reinterpret_cast<Item *>(entries);
        for (int k = 0; k < kKinds; ++k) dst = std::copy(items[k].begin(), items[k].end(), dst);
    } catch (...) {
        return (int)hipErrorOutOfMemory;
    }
    return 0;
}

extern "C" int ct_muon(const ct_muon_matrix *matrices, int64_t count, const int32_t *plan, const int64_t *counts,
                       int32_t dtype, const ct_muon_options *o, void *workspace, int64_t workspace_bytes,
                       int64_t workspace_needed, hipStream_t stream) {
    if (!counts || !o) return -CT_EINVAL_POINTER;
    if (dtype != CT_F32 && dtype != CT_BF16) return -CT_EINVAL_DTYPE;
    if (o->steps < 1 || o->steps > 100 || count < 0) return -CT_EINVAL_SHAPE;
    for (int k = 0; k < kKinds; ++k)
        if (counts[k] < 0 || counts[k] > 0x7fffffff) return -CT_EINVAL_SHAPE;
    if (count == 0) return 0;
    if (!matrices || !plan || (uintptr_t)plan % 16) return -CT_EINVAL_POINTER;
    for (int64_t i = 0; i < count; ++i)
        if (!matrices[i].param || !matrices[i].grad || (o->update && !matrices[i].momentum)) return -CT_EINVAL_POINTER;
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < workspace_needed) return -CT_EINVAL_WORKSPACE;
    Hyper h;
    h.lr = (float)o->lr;
    h.mu = (float)o->momentum;
    h.rest = (float)(1.0 - o->momentum);
    h.keep = (float)(1.0 - o->lr * o->weight_decay);
    h.nesterov = o->nesterov ? 1 : 0;
    h.step = o->update ? 1 : 0;
    h.a = o->a;
    h.b = o->b;
    h.c = o->c;
    h.eps = o->eps;
    const Matrix *mats = static_cast<const Matrix *>(workspace);
    const Item *items[kKinds];
    items[0] = reinterpret_cast<const Item *>(plan);
    for (int k = 1; k < kKinds; ++k) items[k] = items[k - 1] + counts[k - 1];
    double *ws = static_cast<double *>(workspace);
    auto grid = [&](int kind, unsigned y = 1) { return dim3((unsigned)counts[kind], y); };
    const bool half = dtype == CT_BF16;
    int status = 0;
    auto ok = [&]() { return (status = status_of_last_launch()) == 0; };
    for (int64_t i = 0; i < count; i += kTableChunk) {
        TableChunk chunk = {};
        const int n = (int)std::min<int64_t>(kTableChunk, count - i);
        std::copy_n(reinterpret_cast<const Matrix *>(matrices) + i, n, chunk.m);
        muon_table<<<dim3(1), dim3(64), 0, stream>>>(static_cast<Matrix *>(workspace) + i, chunk, n);
        if (!ok()) return status;
    }
    if (counts[kItemsGram]) {
        const auto kernel = half ? muon_gram<uint16_t> : muon_gram<float>;
        kernel<<<grid(kItemsGram), dim3(kGramThreads), 0, stream>>>(mats, items[kItemsGram], h, ws);
        if (!ok()) return status;
    }
    if (counts[kItemsTiles]) {
        if (h.step) {
            const auto kernel = half ? muon_momentum<uint16_t> : muon_momentum<float>;
            kernel<<<grid(kItemsMomentum), dim3(kThreads), 0, stream>>>(mats, items[kItemsMomentum], h);
            if (!ok()) return status;
        }
        const auto kernel = half ? muon_gram_tiles<uint16_t> : muon_gram_tiles<float>;
        kernel<<<grid(kItemsTiles), dim3(kThreads), 0, stream>>>(mats, items[kItemsTiles], h, ws);
        if (!ok()) return status;
    }
    if (counts[kItemsSmall]) {
        muon_small<<<grid(kItemsSmall), dim3(kSmallThreads), 0, stream>>>(mats, items[kItemsSmall], h, ws, o->steps);
        if (!ok()) return status;
    }
    if (counts[kItemsStage]) {
        muon_join<<<grid(kItemsJoin), dim3(kThreads), 0, stream>>>(mats, items[kItemsJoin], h, ws);
        if (!ok()) return status;
        auto stage = [&](const StageOp &op0, const StageOp *op1) {
            muon_stage<<<grid(kItemsStage, op1 ? 2 : 1), dim3(kStageThreads), 0, stream>>>(
                mats, items[kItemsStage], h, ws, op0, op1 ? *op1 : op0);
            return ok();
        };
        int q = kQ;   // the product of the P so far; the first P is the first Q
        for (int i = 0; i < o->steps; ++i) {
            const bool first = i == 0, last = i + 1 == o->steps;
            const int p = first ? kQ : kP, next = q == kQ ? kQ + 1 : kQ;
            if (!stage({kMakeP, kG, kG, p, first && last}, nullptr)) return status;
            const StageOp extend = {kMultiply, p, q, next, last};
            if (!last) {
                if (!stage({kMultiply, p, kG, kT, 0}, first ? nullptr : &extend)) return status;
                if (!stage({kMultiply, p, kT, kG, 0}, nullptr)) return status;
            } else if (!first) {
                if (!stage(extend, nullptr)) return status;
            }
            if (!first) q = next;
        }
    }
    const auto kernel = half ? (h.step ? muon_apply<uint16_t, true> : muon_apply<uint16_t, false>)
                             : (h.step ? muon_apply<float, true> : muon_apply<float, false>);
    kernel<<<grid(kItemsApply), dim3(kApplyThreads), 0, stream>>>(mats, items[kItemsApply], h, ws);
    return status_of_last_launch();
}
