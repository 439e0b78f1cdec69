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
constexpr int kGramTile = 64;   // rows of M per side of a Gram share
constexpr int kCols = 64;       // long-side elements per share of the last product
constexpr int kEntry = 8;       // int32 per plan entry

struct Matrix {                 // ct_muon_matrix
    void *param;
    const void *grad;
    float *momentum;
    int64_t rows, cols;
    int64_t scratch;            // doubles from the workspace's start
    int64_t parts;              // partial Gram tiles of this matrix: first, in tiles of 64 x 64 doubles
    float adjust;
    int32_t splits;
};

struct Item {
    int32_t matrix, i, j, lo, hi, pad0, pad1, pad2;
};

struct Hyper {
    float lr, mu, rest, keep;   // rest = 1 - mu, keep = 1 - lr decay
    int nesterov, step;   // step: 0 = orthogonalize grad into param
    double a, b, c, eps;
};

__device__ __forceinline__ int short_side(const Matrix &m) { return (int)(m.rows < m.cols ? m.rows : m.cols); }
__device__ __forceinline__ int padded(int r) { return (r + kPad - 1) / kPad * kPad; }

template <typename T>
__device__ __forceinline__ float load_elem(const void *p, int64_t i) {
    if constexpr (sizeof(T) == 2) return bf16_to_f32(static_cast<const uint16_t *>(p)[i]);
    else return static_cast<const float *>(p)[i];
}

// Element of M: the gradient, or the step's combination of it with the updated momentum.
template <typename T>
__device__ __forceinline__ float source(const Matrix &m, const Hyper &h, int64_t i) {
    const float g = load_elem<T>(m.grad, i);
    if (!h.step) return g;
    const float v = m.momentum[i];
    return h.nesterov ? __builtin_fmaf(h.mu, v, h.rest * g) : v;
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

// ------------------------------------------------------------------ momentum
template <typename T>
__global__ __launch_bounds__(kThreads) void muon_momentum(const Matrix *matrices, const Item *items, Hyper h) {
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    const int r = short_side(m);
    const int64_t width = m.rows * m.cols / r;
    const int64_t end = (int64_t)it.hi < width ? (int64_t)it.hi * r : width * r;
    for (int64_t i = (int64_t)it.lo * r + threadIdx.x; i < end; i += kThreads)
        m.momentum[i] = __builtin_fmaf(h.mu, m.momentum[i], h.rest * load_elem<T>(m.grad, i));
}

// ------------------------------------------------------------------ Gram matrix
// D[4 i + l / 16][l % 16] for i = 0..3 of A[l % 16][l / 16] B[l / 16][l % 16].
__device__ __forceinline__ f64x4 mfma_f64(double a, double b, f64x4 c) {
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
}

// One 64 x 64 tile (i >= j) of M M^T over the columns lo .. hi - 1: 4 waves of 32 x 32.
template <typename T>
__global__ __launch_bounds__(kThreads) void muon_gram(const Matrix *matrices, const Item *items, Hyper h, double *ws) {
    constexpr int KC = 16, kPitch = KC + 4;
    __shared__ float sa[kGramTile * kPitch], sb[kGramTile * kPitch];
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    const int r = short_side(m), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
    double *dst = ws + (m.parts + it.pad0) * (kGramTile * kGramTile);
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                dst[(wi + 16 * x + 4 * i + (lane >> 4)) * kGramTile + wj + 16 * y + (lane & 15)] = acc[x][y][i];
}

// Buffers of one matrix in the workspace: G, P, T, two Q (doubles) and the final float Q.
__device__ __forceinline__ double *buffer(const Matrix &m, double *ws, int which) {
    const int64_t rp = padded(short_side(m));
    return ws + m.scratch + 2 + which * rp * rp;   // [0] holds 1 / |M|
}
enum { kG = 0, kP = 1, kT = 2, kQ = 3, kFinal = 5 };

// Partial tile that covers element (i, j), i >= j, split s.
__device__ __forceinline__ double part(const Matrix &m, const double *ws, int i, int j, int s) {
    const int ti = i / kGramTile, tj = j / kGramTile;
    return ws[(m.parts + (ti * (ti + 1) / 2 + tj) * (int64_t)m.splits + s) * (kGramTile * kGramTile) +
              (i % kGramTile) * kGramTile + j % kGramTile];
}

// G of a 32 x 32 tile: the partial sums in order, over the squared norm (G's trace, which
// every workgroup sums for itself in one order).
__global__ __launch_bounds__(kThreads) void muon_join(const Matrix *matrices, const Item *items, Hyper h, double *ws) {
    __shared__ double sums[kThreads];
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    const int r = short_side(m), rp = padded(r);
    double trace = 0.0;
    for (int i = threadIdx.x; i < r; i += kThreads)
        for (int s = 0; s < m.splits; ++s) trace += part(m, ws, i, i, s);
    sums[threadIdx.x] = trace;
    __syncthreads();
    for (int n = kThreads / 2; n; n >>= 1) {
        if ((int)threadIdx.x < n) sums[threadIdx.x] += sums[threadIdx.x + n];
        __syncthreads();
    }
    const double norm = sqrt(sums[0]), inv = 1.0 / (norm < h.eps ? h.eps : norm);
    if (it.i == 0 && threadIdx.x == 0) ws[m.scratch] = inv;
    double *g = buffer(m, ws, kG);
    for (int e = threadIdx.x; e < kPad * kPad; e += kThreads) {
        const int i = it.i * kPad + e / kPad, j = it.j * kPad + e % kPad;
        if (i < j) continue;
        double v = 0.0;
        if (i < r)
            for (int s = 0; s < m.splits; ++s) v += part(m, ws, i, j, s);
        v *= inv * inv;
        g[(int64_t)i * rp + j] = v;
        g[(int64_t)j * rp + i] = v;
    }
}

// ------------------------------------------------------------------ r x r products
enum StageKind { kMakeP = 0, kMultiply = 1 };

struct StageOp {
    int kind, left, right, dst, last;
};

// One 32 x 32 tile (i >= j) of left right, both symmetric and commuting, so their product is
// symmetric too and the tile's mirror image is its transpose. kMakeP: a I + b G + c G G.
__global__ __launch_bounds__(kThreads) void muon_stage(const Matrix *matrices, const Item *items, Hyper h, double *ws,
                                                      StageOp op0, StageOp op1) {
    constexpr int KC = 32, kPitch = KC + 4;
    __shared__ double sa[kPad * kPitch], sb[kPad * kPitch];
    const StageOp op = blockIdx.y ? op1 : op0;
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    const int r = short_side(m), rp = padded(r), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double *left = buffer(m, ws, op.left) + (int64_t)it.i * kPad * rp;
    const double *right = buffer(m, ws, op.right) + (int64_t)it.j * kPad * rp;
    const int wi = (wave >> 1) * 16, wj = (wave & 1) * 16;
    f64x4 acc = {};
    for (int k0 = 0; k0 < rp; k0 += KC) {
        __syncthreads();
        for (int e = threadIdx.x; e < kPad * KC; e += kThreads) {
            sa[e / KC * kPitch + e % KC] = left[(int64_t)(e / KC) * rp + k0 + e % KC];
            sb[e / KC * kPitch + e % KC] = right[(int64_t)(e / KC) * rp + k0 + e % KC];
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < KC; s += 4)
            acc = mfma_f64(sa[(wi + (lane & 15)) * kPitch + s + (lane >> 4)],
                           sb[(wj + (lane & 15)) * kPitch + s + (lane >> 4)], acc);
    }
    const double inv = op.last ? ws[m.scratch] : 1.0;
    double *dst = buffer(m, ws, op.dst);
    float *final = reinterpret_cast<float *>(buffer(m, ws, kFinal));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int i = it.i * kPad + wi + 4 * e + (lane >> 4), j = it.j * kPad + wj + (lane & 15);
        if (i < j) continue;
        double v = acc[e];
        if (op.kind == kMakeP) {
            v = h.c * v + h.b * left[(int64_t)(i - it.i * kPad) * rp + j];
            if (i == j && i < r) v += h.a;
        }
        const int64_t x = (int64_t)i * rp + j, y = (int64_t)j * rp + i;
        if (op.last) {
            final[x] = final[y] = (float)(v * inv);
        } else {
            dst[x] = v;
            dst[y] = v;
        }
    }
}

// ------------------------------------------------------------------ the last product
// 64 elements of the long side, all of the short side in blocks of 128: 4 waves of 32 x 64
// (wide) or 64 x 32 (tall), v_mfma_f32_32x32x2.
template <typename T>
__global__ __launch_bounds__(kThreads) void muon_apply(const Matrix *matrices, const Item *items, Hyper h, double *ws) {
    constexpr int KC = 32, kPitch = KC + 1;
    __shared__ float sx[kCols * kPitch];   // [long][short]
    const Item it = items[blockIdx.x];
    const Matrix m = matrices[it.matrix];
    const int r = short_side(m), rp = padded(r), lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const bool tall = m.rows > m.cols;
    const int64_t width = tall ? m.rows : m.cols, col0 = (int64_t)it.i * kCols;
    const float *q = reinterpret_cast<const float *>(buffer(m, ws, kFinal));
    for (int r0 = 0; r0 < rp; r0 += 128) {
        const int row = r0 + wave * 32 + (lane & 31);
        f32x16 acc[2] = {};
        for (int k0 = 0; k0 < rp; k0 += KC) {
            __syncthreads();
            for (int e = threadIdx.x; e < kCols * KC; e += kThreads) {
                const int c = tall ? e / KC : e % kCols, k = tall ? e % KC : e / kCols;
                float v = 0.0f;
                if (k0 + k < r && col0 + c < width)
                    v = source<T>(m, h, tall ? (col0 + c) * r + k0 + k : (int64_t)(k0 + k) * m.cols + col0 + c);
                sx[c * kPitch + k] = v;
            }
            __syncthreads();
            if (r0 + wave * 32 < rp) {
#pragma unroll
                for (int k = 0; k < KC; k += 2) {
                    const float w = q[(int64_t)(k0 + k + half) * rp + row];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        const float x = sx[(32 * t + (lane & 31)) * kPitch + k + half];
                        acc[t] = tall ? __builtin_amdgcn_mfma_f32_32x32x2f32(x, w, acc[t], 0, 0, 0)
                                      : __builtin_amdgcn_mfma_f32_32x32x2f32(w, x, acc[t], 0, 0, 0);
                    }
                }
            }
        }
        if (r0 + wave * 32 >= rp) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int down = 8 * (i >> 2) + 4 * half + (i & 3), across = lane & 31;
                const int s = r0 + wave * 32 + (tall ? across : down);
                const int64_t l = col0 + 32 * t + (tall ? down : across);
                if (s >= r || l >= width) continue;
                const int64_t at = tall ? l * r + s : (int64_t)s * m.cols + l;
                float v = acc[t][i];
                if (h.step) {
                    const float p = load_elem<T>(m.param, at);
                    v = __builtin_fmaf(-h.lr * m.adjust, v, p * h.keep);
                }
                if constexpr (sizeof(T) == 2) static_cast<uint16_t *>(m.param)[at] = bf16_bits(v);
                else static_cast<float *>(m.param)[at] = v;
            }
    }
}

// ------------------------------------------------------------------ host side
constexpr int64_t kMaxShort = 16384, kMaxLong = (int64_t)1 << 30;

struct Shape {
    int64_t r, width, rp, pairs, splits;
};

bool shape_of(int64_t rows, int64_t cols, Shape &s) {
    if (rows <= 0 || cols <= 0) return false;
    s.r = std::min(rows, cols);
    s.width = std::max(rows, cols);
    if (s.r > kMaxShort || s.width > kMaxLong) return false;
    s.rp = cdiv(s.r, kPad) * kPad;
    const int64_t tiles = cdiv(s.r, kGramTile);
    s.pairs = tiles * (tiles + 1) / 2;
    s.splits = std::max<int64_t>(1, std::min<int64_t>(cdiv(s.width, 512), 32));
    return true;
}

int64_t scratch_doubles(const Shape &s) { return 2 + 5 * s.rp * s.rp + s.rp * s.rp / 2; }

int status_of_last_launch() {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : (int)e;
}

}  // namespace
}  // namespace ct

using namespace ct;

static_assert(kGramTile * kGramTile * sizeof(double) == 32768 && sizeof(TableChunk) < 4000, "table");
static_assert(sizeof(Matrix) == sizeof(ct_muon_matrix), "ct_muon_matrix");

extern "C" int ct_muon_plan(ct_muon_matrix *matrices, int64_t count, int32_t *entries, int64_t capacity,
                            int64_t *counts, int64_t *workspace_bytes) {
    if (count < 0 || count > 0x7fffffff) return -CT_EINVAL_SHAPE;
    if (!counts || !workspace_bytes || (count && !matrices)) return -CT_EINVAL_POINTER;
    try {
        std::vector<Item> gram, stage, apply;
        int64_t doubles = 0, parts = 0;
        for (int64_t i = 0; i < count; ++i) {
            Shape s;
            if (!shape_of(matrices[i].rows, matrices[i].cols, s)) return -CT_EINVAL_SHAPE;
            matrices[i].parts = parts;
            matrices[i].splits = (int32_t)s.splits;
            parts += s.pairs * s.splits;
            const int64_t step = cdiv(cdiv(s.width, s.splits), 16) * 16, tiles = cdiv(s.r, kGramTile);
            int32_t slot = 0;
            for (int64_t a = 0; a < tiles; ++a)
                for (int64_t b = 0; b <= a; ++b)
                    for (int64_t k = 0; k < s.splits; ++k)
                        gram.push_back({(int32_t)i, (int32_t)a, (int32_t)b, (int32_t)std::min(s.width, k * step),
                                        (int32_t)std::min(s.width, (k + 1) * step), slot++, 0, 0});
            for (int64_t a = 0; a < s.rp / kPad; ++a)
                for (int64_t b = 0; b <= a; ++b) stage.push_back({(int32_t)i, (int32_t)a, (int32_t)b, 0, 0, 0, 0, 0});
            for (int64_t c = 0; c < cdiv(s.width, kCols); ++c)
                apply.push_back({(int32_t)i, (int32_t)c, 0, (int32_t)(c * kCols),
                                 (int32_t)std::min(s.width, (c + 1) * kCols), 0, 0, 0});
        }
        for (int64_t i = 0; i < count; ++i) matrices[i].parts += cdiv(count * (int64_t)sizeof(Matrix), 32768);
        // the table first, then the partial tiles, then each matrix's buffers
        doubles = (parts + cdiv(count * (int64_t)sizeof(Matrix), 32768)) * kGramTile * kGramTile;
        for (int64_t i = 0; i < count; ++i) {
            Shape s;
            shape_of(matrices[i].rows, matrices[i].cols, s);
            matrices[i].scratch = doubles;
            doubles += scratch_doubles(s);
        }
        counts[0] = (int64_t)gram.size();
        counts[1] = (int64_t)stage.size();
        counts[2] = (int64_t)apply.size();
        *workspace_bytes = doubles * (int64_t)sizeof(double);
        for (int i = 0; i < 3; ++i)
            if (counts[i] > 0x7fffffff / kThreads) return -CT_EINVAL_SHAPE;
        if (!entries) return 0;
        if (capacity < counts[0] + counts[1] + counts[2]) return -CT_EINVAL_WORKSPACE;
        Item *dst = reinterpret_cast<Item *>(entries);
        dst = std::copy(gram.begin(), gram.end(), dst);
        dst = std::copy(stage.begin(), stage.end(), dst);
        std::copy(apply.begin(), apply.end(), dst);
    } catch (...) {
        return (int)hipErrorOutOfMemory;
    }
    return 0;
}

extern "C" int ct_muon(const ct_muon_matrix *matrices, int64_t count, const int32_t *plan, const int64_t *counts, int32_t dtype,
                       const ct_muon_options *o, void *workspace, int64_t workspace_bytes, int64_t workspace_needed,
                       hipStream_t stream) {
    if (!counts || !o) return -CT_EINVAL_POINTER;
    if (dtype != CT_F32 && dtype != CT_BF16) return -CT_EINVAL_DTYPE;
    if (o->steps < 1 || o->steps > 100 || counts[0] < 0 || counts[1] < 0 || counts[2] < 0 || counts[0] > 0x7fffffff ||
        counts[1] > 0x7fffffff || counts[2] > 0x7fffffff)
        return -CT_EINVAL_SHAPE;
    if (count <= 0 || counts[0] == 0) return count < 0 ? -CT_EINVAL_SHAPE : 0;
    if (!matrices || !plan || (uintptr_t)plan % 16) return -CT_EINVAL_POINTER;
    for (int64_t i = 0; i < count; ++i)
        if (!matrices[i].param || !matrices[i].grad || (o->update && !matrices[i].momentum)) return -CT_EINVAL_POINTER;
    if (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < workspace_needed) return -CT_EINVAL_WORKSPACE;
    const Matrix *mats = static_cast<const Matrix *>(workspace);
    const Item *gram = reinterpret_cast<const Item *>(plan), *stage = gram + counts[0], *apply = stage + counts[1];
    double *ws = static_cast<double *>(workspace);
    Hyper h;
    h.lr = (float)o->lr;
    h.keep = (float)(1.0 - o->lr * o->weight_decay);
    h.mu = (float)o->momentum;
    h.rest = (float)(1.0 - o->momentum);
    h.nesterov = o->nesterov ? 1 : 0;
    h.step = o->update ? 1 : 0;
    h.a = o->a;
    h.b = o->b;
    h.c = o->c;
    h.eps = o->eps;
    const dim3 threads(kThreads);
    int status = 0;
    auto ok = [&]() { return (status = status_of_last_launch()) == 0; };
    for (int64_t i = 0; i < count; i += kTableChunk) {
        TableChunk chunk;
        const int n = (int)std::min<int64_t>(kTableChunk, count - i);
        std::copy_n(reinterpret_cast<const Matrix *>(matrices) + i, n, chunk.m);
        muon_table<<<dim3(1), dim3(64), 0, stream>>>(static_cast<Matrix *>(workspace) + i, chunk, n);
        if (!ok()) return status;
    }
    if (h.step) {
        if (dtype == CT_BF16) muon_momentum<uint16_t><<<dim3((unsigned)counts[2]), threads, 0, stream>>>(mats, apply, h);
        else muon_momentum<float><<<dim3((unsigned)counts[2]), threads, 0, stream>>>(mats, apply, h);
        if (!ok()) return status;
    }
    if (dtype == CT_BF16) muon_gram<uint16_t><<<dim3((unsigned)counts[0]), threads, 0, stream>>>(mats, gram, h, ws);
    else muon_gram<float><<<dim3((unsigned)counts[0]), threads, 0, stream>>>(mats, gram, h, ws);
    if (!ok()) return status;
    muon_join<<<dim3((unsigned)counts[1]), threads, 0, stream>>>(mats, stage, h, ws);
    if (!ok()) return status;
    const dim3 one((unsigned)counts[1], 1), two((unsigned)counts[1], 2);
    int q = kP;   // the product of the P so far
    for (int i = 0; i < o->steps; ++i) {
        const bool first = i == 0, last = i + 1 == o->steps;
        // the first P is the first Q and is not overwritten before the second step has read it
        const int p = first ? kQ : kP;
        muon_stage<<<one, threads, 0, stream>>>(mats, stage, h, ws, {kMakeP, kG, kG, p, first && last}, {});
        if (!ok()) return status;
        const int next = q == kQ ? kQ + 1 : kQ;
        const StageOp extend = {kMultiply, p, q, next, last}, shift = {kMultiply, p, kG, kT, 0};
        if (!last) {
            muon_stage<<<first ? one : two, threads, 0, stream>>>(mats, stage, h, ws, shift, extend);
            if (!ok()) return status;
            muon_stage<<<one, threads, 0, stream>>>(mats, stage, h, ws, {kMultiply, p, kT, kG, 0}, {});
        } else if (!first) {
            muon_stage<<<one, threads, 0, stream>>>(mats, stage, h, ws, extend, {});
        }
        if (!ok()) return status;
        q = first ? kQ : next;
    }
    if (dtype == CT_BF16) muon_apply<uint16_t><<<dim3((unsigned)counts[2]), threads, 0, stream>>>(mats, apply, h, ws);
    else muon_apply<float><<<dim3((unsigned)counts[2]), threads, 0, stream>>>(mats, apply, h, ws);
    return status_of_last_launch();
}
