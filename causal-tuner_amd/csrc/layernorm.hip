// Row-wise layer normalization on gfx950, forward and backward, all in float32:
//
//   forward   mean = sum(x) / width, rstd = 1 / sqrt(sum((x - mean)^2) / width + eps)
//             y = (x - mean) rstd w + bias                                  (rounded once)
//   backward  g = dy w, n = (x - mean) rstd
//             dx = rstd (g - sum(g) / width - n sum(g n) / width)
//             dw = sum over rows of dy n, dbias = sum over rows of dy
//
// Bound by HBM: the forward reads x and writes y, the backward reads x and dy and writes dx. A row
// is held in the registers of its team of threads (a wave, 256 or 1024 threads), so it is read once;
// the variance is of the differences from the mean, in a second pass over the registers. In the
// backward each team walks rows with fixed columns per thread and sums dw and dbias in registers
// on the way; the teams' sums, one row of the workspace each, are joined in a fixed order by a
// second launch. Rows wider than the registers of a team take kernels that read them again.
// 16384 x 4096 bf16: forward 45 to 60 us (5.9 to 4.5 TB/s, by what the last-level cache holds), backward 83
// (4.9 TB/s) and 4 for the joining; 30000 x 1023 float32 backward 87 us (4.2 TB/s).

#include <math.h>

#include "common.hpp"

namespace ct {
namespace {

template <int DT>
struct Element {
    static constexpr int kSize = DT == CT_F32 ? 4 : 2, kPer = 16 / kSize;
};

template <int DT>
__device__ __forceinline__ float load1(const void *p, int64_t i) {
    if constexpr (DT == CT_F32) return static_cast<const float *>(p)[i];
    else if constexpr (DT == CT_BF16) return bf16_to_f32(static_cast<const uint16_t *>(p)[i]);
    else return f16_to_f32(static_cast<const uint16_t *>(p)[i]);
}
template <int DT>
__device__ __forceinline__ void store1(void *p, int64_t i, float v) {
    if constexpr (DT == CT_F32) static_cast<float *>(p)[i] = v;
    else static_cast<uint16_t *>(p)[i] = DT == CT_BF16 ? bf16_bits(v) : f16_bits(v);
}
__device__ __forceinline__ float load_any(const void *p, int dtype, int64_t i) {
    return dtype == CT_F32 ? load1<CT_F32>(p, i) : dtype == CT_BF16 ? load1<CT_BF16>(p, i) : load1<CT_F16>(p, i);
}
__device__ __forceinline__ void store_any(void *p, int dtype, int64_t i, float v) {
    if (dtype == CT_F32) store1<CT_F32>(p, i, v);
    else if (dtype == CT_BF16) store1<CT_BF16>(p, i, v);
    else store1<CT_F16>(p, i, v);
}

// A thread's chunk of a row: E values, as one 16-byte access (E > 1) or one element.
template <int DT, int E>
struct Chunk {
    uint4 raw;
    __device__ __forceinline__ void load(const void *row, int64_t c) {
        if constexpr (E > 1) raw = *reinterpret_cast<const uint4 *>(static_cast<const char *>(row) + c * Element<DT>::kSize);
        else raw.x = __builtin_bit_cast(uint32_t, load1<DT>(row, c));
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (E == 1) return __builtin_bit_cast(float, raw.x);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (DT == CT_F32) return __builtin_bit_cast(float, w[e]);
        const uint16_t h = (uint16_t)(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu);
        return DT == CT_BF16 ? bf16_to_f32(h) : f16_to_f32(h);
    }
};
template <int DT, int E>
__device__ __forceinline__ void store_chunk(void *row, int64_t c, const float *v) {
    if constexpr (E == 1) {
        store1<DT>(row, c, v[0]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == CT_F32) w[i] = __builtin_bit_cast(uint32_t, v[i]);
            else if constexpr (DT == CT_BF16) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
            else w[i] = (uint32_t)f16_bits(v[2 * i]) | (uint32_t)f16_bits(v[2 * i + 1]) << 16;
        }
        *reinterpret_cast<uint4 *>(static_cast<char *>(row) + c * Element<DT>::kSize) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}
// E values of a vector of any of the types (16-byte aligned where E > 1).
template <int E>
__device__ __forceinline__ void load_vector(const void *p, int dtype, int64_t c, float *v) {
    if constexpr (E == 1) {
        v[0] = load_any(p, dtype, c);
    } else if (dtype == CT_F32) {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + c + e);
            v[e] = f.x, v[e + 1] = f.y, v[e + 2] = f.z, v[e + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const uint2 h = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + c + e);
            const uint32_t w[2] = {h.x, h.y};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint16_t b = (uint16_t)(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xffffu);
                v[e + i] = dtype == CT_BF16 ? bf16_to_f32(b) : f16_to_f32(b);
            }
        }
    }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// Sums of N values over the team, the waves' in order. Two calls in a row take different `lds`.
template <int TEAM, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float *lds) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
    if constexpr (TEAM > 64) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) lds[wave * N + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < TEAM / 64; ++w) v[i] += lds[w * N + i];
        }
    }
}

template <int DT, int E, int TEAM, int C>
__global__ __launch_bounds__(TEAM > 256 ? TEAM : 256) void forward_kernel(const void *__restrict__ x,
                                                                          const void *__restrict__ w,
                                                                          const void *__restrict__ bias, int w_dtype,
                                                                          void *__restrict__ y, float *__restrict__ mean_out,
                                                                          float *__restrict__ rstd_out, int64_t rows,
                                                                          int64_t width, float eps) {
    constexpr int THREADS = TEAM > 256 ? TEAM : 256;
    __shared__ float lds[2][TEAM / 64];
    const int t = threadIdx.x % TEAM;
    const int64_t row = (int64_t)blockIdx.x * (THREADS / TEAM) + threadIdx.x / TEAM;
    if (TEAM == 64 && row >= rows) return;   // a whole wave; larger teams have a workgroup per row
    const char *in = static_cast<const char *>(x) + row * width * Element<DT>::kSize;
    Chunk<DT, E> v[C];
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int64_t c = ((int64_t)i * TEAM + t) * E;
        if (c < width) {
            v[i].load(in, c);
#pragma unroll
            for (int e = 0; e < E; ++e) s[0] += v[i].get(e);
        }
    }
    team_sum<TEAM>(s, lds[0]);
    const float mean = s[0] / (float)width;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i)
        if (((int64_t)i * TEAM + t) * E < width)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float d = v[i].get(e) - mean;
                s[0] += d * d;
            }
    team_sum<TEAM>(s, lds[1]);
    const float rstd = 1.f / sqrtf(s[0] / (float)width + eps);
    char *out = static_cast<char *>(y) + row * width * Element<DT>::kSize;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int64_t c = ((int64_t)i * TEAM + t) * E;
        if (c >= width) continue;
        float o[E], k[E];
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = (v[i].get(e) - mean) * rstd;
        if (w) {
            load_vector<E>(w, w_dtype, c, k);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= k[e];
        }
        if (bias) {
            load_vector<E>(bias, w_dtype, c, k);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += k[e];
        }
        store_chunk<DT, E>(out, c, o);
    }
    if (mean_out && t == 0) {
        mean_out[row] = mean;
        rstd_out[row] = rstd;
    }
}

// Teams walk rows team, team + teams, ...; `partial` [team][2][width] takes their sums of dw and dbias.
template <int DT, int E, int TEAM, int C>
__global__ __launch_bounds__(TEAM > 256 ? TEAM : 256) void backward_kernel(const void *__restrict__ x,
                                                                           const void *__restrict__ w, int w_dtype,
                                                                           const float *__restrict__ mean,
                                                                           const float *__restrict__ rstd, const void *dy,
                                                                           void *dx, float *__restrict__ partial,
                                                                           int64_t rows, int64_t width) {
    constexpr int THREADS = TEAM > 256 ? TEAM : 256, TEAMS = THREADS / TEAM;
    __shared__ float lds[2][2 * TEAM / 64];
    const int t = threadIdx.x % TEAM;
    const int64_t team = (int64_t)blockIdx.x * TEAMS + threadIdx.x / TEAM, teams = (int64_t)gridDim.x * TEAMS;
    float k[C][E], sum_w[C][E], sum_b[C][E];
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int64_t c = ((int64_t)i * TEAM + t) * E;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            k[i][e] = 1.f;
            sum_w[i][e] = sum_b[i][e] = 0.f;
        }
        if (w && c < width) load_vector<E>(w, w_dtype, c, k[i]);
    }
    Chunk<DT, E> vx[C], vy[C];
    const auto load = [&](int64_t row) {
        const int64_t base = row * width * Element<DT>::kSize;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int64_t c = ((int64_t)i * TEAM + t) * E;
            if (c < width) {
                vx[i].load(static_cast<const char *>(x) + base, c);
                vy[i].load(static_cast<const char *>(dy) + base, c);
            }
        }
    };
    const float scale = 1.f / (float)width;
    float m = 0.f, r = 0.f;
    if (team < rows) {
        load(team);
        m = mean[team];
        r = rstd[team];
    }
    int turn = 0;
    for (int64_t row = team; row < rows; row += teams, turn ^= 1) {
        Chunk<DT, E> cx[C], cy[C];
        const float now_m = m, now = r;
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < C; ++i) {
            cx[i] = vx[i];
            cy[i] = vy[i];
        }
        if (row + teams < rows) {   // the next row's loads run over this one's sums
            load(row + teams);
            m = mean[row + teams];
            r = rstd[row + teams];
        }
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (((int64_t)i * TEAM + t) * E < width)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const float n = (cx[i].get(e) - now_m) * now, d = cy[i].get(e), g = d * k[i][e];
                    s[0] += g;
                    s[1] += g * n;
                    sum_w[i][e] += d * n;
                    sum_b[i][e] += d;
                }
        if (!dx) continue;
        team_sum<TEAM>(s, lds[turn]);
        const float a = s[0] * scale, b = s[1] * scale;
        char *out = static_cast<char *>(dx) + row * width * Element<DT>::kSize;
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int64_t c = ((int64_t)i * TEAM + t) * E;
            if (c >= width) continue;
            float o[E];
#pragma unroll
            for (int e = 0; e < E; ++e)
                o[e] = now * (cy[i].get(e) * k[i][e] - a - (cx[i].get(e) - now_m) * now * b);
            store_chunk<DT, E>(out, c, o);
        }
    }
    if (!partial) return;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        const int64_t c = ((int64_t)i * TEAM + t) * E;
        if (c >= width) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            partial[team * 2 * width + c + e] = sum_w[i][e];
            partial[(team * 2 + 1) * width + c + e] = sum_b[i][e];
        }
    }
}

// dw (blockIdx.y 0) or dbias (1) of 64 columns: sixteen runs of the partial rows, joined in order.
__global__ __launch_bounds__(1024) void join_kernel(const float *__restrict__ partial, int64_t count, int64_t width,
                                                    void *__restrict__ dw, void *__restrict__ dbias, int w_dtype) {
    __shared__ float lds[16][64];
    void *out = blockIdx.y ? dbias : dw;
    if (!out) return;
    const int col = threadIdx.x & 63, run = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + col, per = cdiv(count, 16);
    float sum = 0.f;
    if (c < width) {
        const int64_t end = (run + 1) * per < count ? (run + 1) * per : count;
#pragma unroll 8
        for (int64_t i = run * per; i < end; ++i) sum += partial[(i * 2 + blockIdx.y) * width + c];
    }
    lds[run][col] = sum;
    __syncthreads();
    if (run == 0 && c < width) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += lds[i][col];
        store_any(out, w_dtype, c, sum);
    }
}

// ------------------------------------------------------------------------- rows of any width
template <int DT>
__global__ __launch_bounds__(1024) void forward_wide(const void *__restrict__ x, const void *__restrict__ w,
                                                     const void *__restrict__ bias, int w_dtype, void *__restrict__ y,
                                                     float *__restrict__ mean_out, float *__restrict__ rstd_out,
                                                     int64_t width, float eps) {
    __shared__ float lds[2][16];
    const int64_t base = (int64_t)blockIdx.x * width;
    float s[1] = {0.f};
    for (int64_t c = threadIdx.x; c < width; c += 1024) s[0] += load1<DT>(x, base + c);
    team_sum<1024>(s, lds[0]);
    const float mean = s[0] / (float)width;
    s[0] = 0.f;
    for (int64_t c = threadIdx.x; c < width; c += 1024) {
        const float d = load1<DT>(x, base + c) - mean;
        s[0] += d * d;
    }
    team_sum<1024>(s, lds[1]);
    const float rstd = 1.f / sqrtf(s[0] / (float)width + eps);
    for (int64_t c = threadIdx.x; c < width; c += 1024) {
        float o = (load1<DT>(x, base + c) - mean) * rstd;
        if (w) o *= load_any(w, w_dtype, c);
        if (bias) o += load_any(bias, w_dtype, c);
        store1<DT>(y, base + c, o);
    }
    if (mean_out && threadIdx.x == 0) {
        mean_out[blockIdx.x] = mean;
        rstd_out[blockIdx.x] = rstd;
    }
}
template <int DT>
__global__ __launch_bounds__(1024) void backward_wide(const void *__restrict__ x, const void *__restrict__ w, int w_dtype,
                                                      const float *__restrict__ mean, const float *__restrict__ rstd,
                                                      const void *dy, void *dx, int64_t width) {
    __shared__ float lds[32];
    const int64_t base = (int64_t)blockIdx.x * width;
    const float m = mean[blockIdx.x], r = rstd[blockIdx.x];
    float s[2] = {0.f, 0.f};
    for (int64_t c = threadIdx.x; c < width; c += 1024) {
        const float g = load1<DT>(dy, base + c) * (w ? load_any(w, w_dtype, c) : 1.f);
        s[0] += g;
        s[1] += g * ((load1<DT>(x, base + c) - m) * r);
    }
    team_sum<1024>(s, lds);
    const float a = s[0] / (float)width, b = s[1] / (float)width;
    for (int64_t c = threadIdx.x; c < width; c += 1024) {
        const float g = load1<DT>(dy, base + c) * (w ? load_any(w, w_dtype, c) : 1.f);
        store1<DT>(dx, base + c, r * (g - a - (load1<DT>(x, base + c) - m) * r * b));
    }
}
// The columns' sums over rows blockIdx.y, + gridDim.y, ...
template <int DT>
__global__ __launch_bounds__(256) void columns_wide(const void *__restrict__ x, const void *__restrict__ dy,
                                                    const float *__restrict__ mean, const float *__restrict__ rstd,
                                                    float *__restrict__ partial, int64_t rows, int64_t width) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= width) return;
    float sum_w = 0.f, sum_b = 0.f;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const float d = load1<DT>(dy, row * width + c);
        sum_w += d * ((load1<DT>(x, row * width + c) - mean[row]) * rstd[row]);
        sum_b += d;
    }
    partial[(int64_t)blockIdx.y * 2 * width + c] = sum_w;
    partial[((int64_t)blockIdx.y * 2 + 1) * width + c] = sum_b;
}

bool aligned(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// The smallest of the teams and chunks per thread that hold a row. Rows that 16-byte accesses do not fit
// (chunks of one element) take many chunks to a thread, so that as many bytes are under way:
// 30000 x 1023 float32 on teams of 256 and 1024 with one to four chunks ran at 3.3 TB/s forward and 2.3 backward.
struct Shape {
    int team, chunks;   // team 0: rows wider than the registers
};
template <int N>
Shape smallest(const Shape (&shapes)[N], int64_t units) {
    for (const Shape s : shapes)
        if (units <= (int64_t)s.team * s.chunks) return s;
    return Shape{0, 0};
}
constexpr Shape kForwardWide[] = {{64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {1024, 2}, {1024, 8}};
constexpr Shape kForwardSingle[] = {{64, 1}, {64, 4}, {64, 16}, {256, 16}, {1024, 16}};
constexpr Shape kBackwardWide[] = {{64, 1}, {64, 2}, {256, 1}, {256, 2}, {1024, 1}, {1024, 2}};
constexpr Shape kBackwardSingle[] = {{64, 1}, {64, 4}, {64, 16}, {256, 16}, {1024, 16}};
Shape forward_shape(int64_t units, bool vec) { return vec ? smallest(kForwardWide, units) : smallest(kForwardSingle, units); }
Shape backward_shape(int64_t units, bool vec) { return vec ? smallest(kBackwardWide, units) : smallest(kBackwardSingle, units); }
int64_t backward_teams(Shape s, int64_t rows) {
    if (s.team == 0) return rows < 64 ? rows : 64;
    const int64_t per = s.team == 64 ? 4 : 1, most = s.team == 1024 ? 256 : 512;   // workgroups (twice as many: 12% slower)
    const int64_t blocks = cdiv(rows, per);
    return (blocks < most ? blocks : most) * per;
}
int64_t units_of(int64_t width, int dtype, bool vec) {
    return vec ? cdiv(width, dtype == CT_F32 ? 4 : 8) : width;
}

template <int DT, int E>
hipError_t launch_forward(const void *x, const void *w, const void *bias, int w_dtype, void *y, float *mean, float *rstd,
                          int64_t rows, int64_t width, float eps, hipStream_t stream) {
    const Shape s = forward_shape(cdiv(width, E), E > 1);
    const auto is = [&](int team, int chunks) { return s.team == team && s.chunks == chunks; };
    const auto run = [&](auto kernel) {
        kernel<<<dim3((unsigned)(s.team == 64 ? cdiv(rows, 4) : rows)), dim3(s.team > 256 ? s.team : 256), 0, stream>>>(
            x, w, bias, w_dtype, y, mean, rstd, rows, width, eps);
    };
    if (is(64, 1)) run(forward_kernel<DT, E, 64, 1>);
    else if (is(64, 4)) run(forward_kernel<DT, E, 64, 4>);
    else if (s.team && E > 1) {
        if constexpr (E > 1) {
            if (is(64, 2)) run(forward_kernel<DT, E, 64, 2>);
            else if (is(256, 2)) run(forward_kernel<DT, E, 256, 2>);
            else if (is(256, 4)) run(forward_kernel<DT, E, 256, 4>);
            else if (is(1024, 2)) run(forward_kernel<DT, E, 1024, 2>);
            else run(forward_kernel<DT, E, 1024, 8>);
        }
    } else if (s.team) {
        if constexpr (E == 1) {
            if (is(64, 16)) run(forward_kernel<DT, E, 64, 16>);
            else if (is(256, 16)) run(forward_kernel<DT, E, 256, 16>);
            else run(forward_kernel<DT, E, 1024, 16>);
        }
    }
    else forward_wide<DT><<<dim3((unsigned)rows), dim3(1024), 0, stream>>>(x, w, bias, w_dtype, y, mean, rstd, width, eps);
    return hipGetLastError();
}

template <int DT, int E>
hipError_t launch_backward(const void *x, const void *w, int w_dtype, const float *mean, const float *rstd, const void *dy,
                           void *dx, float *partial, int64_t teams, int64_t rows, int64_t width, hipStream_t stream) {
    const Shape s = backward_shape(cdiv(width, E), E > 1);
    const auto is = [&](int team, int chunks) { return s.team == team && s.chunks == chunks; };
    const auto run = [&](auto kernel) {
        kernel<<<dim3((unsigned)(s.team == 64 ? teams / 4 : teams)), dim3(s.team > 256 ? s.team : 256), 0, stream>>>(
            x, w, w_dtype, mean, rstd, dy, dx, partial, rows, width);
    };
    if (is(64, 1)) run(backward_kernel<DT, E, 64, 1>);
    else if (s.team && E > 1) {
        if constexpr (E > 1) {
            if (is(64, 2)) run(backward_kernel<DT, E, 64, 2>);
            else if (is(256, 1)) run(backward_kernel<DT, E, 256, 1>);
            else if (is(256, 2)) run(backward_kernel<DT, E, 256, 2>);
            else if (is(1024, 1)) run(backward_kernel<DT, E, 1024, 1>);
            else run(backward_kernel<DT, E, 1024, 2>);
        }
    } else if (s.team) {
        if constexpr (E == 1) {
            if (is(64, 4)) run(backward_kernel<DT, E, 64, 4>);
            else if (is(64, 16)) run(backward_kernel<DT, E, 64, 16>);
            else if (is(256, 16)) run(backward_kernel<DT, E, 256, 16>);
            else run(backward_kernel<DT, E, 1024, 16>);
        }
    }
    else {
        // the columns' sums first: dx may be dy itself
        if (partial) {
            columns_wide<DT><<<dim3((unsigned)cdiv(width, 256), (unsigned)teams), dim3(256), 0, stream>>>(
                x, dy, mean, rstd, partial, rows, width);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        if (dx) backward_wide<DT><<<dim3((unsigned)rows), dim3(1024), 0, stream>>>(x, w, w_dtype, mean, rstd, dy, dx, width);
    }
    return hipGetLastError();
}

bool known(int dtype) { return dtype == CT_F32 || dtype == CT_F16 || dtype == CT_BF16; }

}  // namespace
}  // namespace ct

using namespace ct;

extern "C" int ct_layer_norm_forward(const void *x, int32_t x_dtype, const void *w, const void *bias, int32_t w_dtype,
                                     void *y, float *mean, float *rstd, int64_t rows, int64_t width, double eps,
                                     hipStream_t stream) {
    if (rows < 0 || rows > 0x7fffffff || width <= 0 || width > 0x7fffffff || !(eps >= 0)) return -CT_EINVAL_SHAPE;
    if (!known(x_dtype) || ((w || bias) && !known(w_dtype))) return -CT_EINVAL_DTYPE;
    if (rows == 0) return 0;
    if (!x || !y || !mean != !rstd) return -CT_EINVAL_POINTER;
    const bool vec = aligned(x) && aligned(y) && aligned(w) && aligned(bias) && width % (x_dtype == CT_F32 ? 4 : 8) == 0;
    hipError_t e = hipSuccess;
    // A launch holds fewer than 2^32 threads, 1024 a row at most.
    for (int64_t row = 0, most = 1 << 21; row < rows && e == hipSuccess; row += most) {
        const int64_t count = rows - row < most ? rows - row : most, at = row * width * (x_dtype == CT_F32 ? 4 : 2);
        const auto run = [&](auto launch) {
            return launch(static_cast<const char *>(x) + at, w, bias, w_dtype, static_cast<char *>(y) + at,
                          mean ? mean + row : nullptr, rstd ? rstd + row : nullptr, count, width, (float)eps, stream);
        };
        if (x_dtype == CT_F32) e = vec ? run(launch_forward<CT_F32, 4>) : run(launch_forward<CT_F32, 1>);
        else if (x_dtype == CT_BF16) e = vec ? run(launch_forward<CT_BF16, 8>) : run(launch_forward<CT_BF16, 1>);
        else e = vec ? run(launch_forward<CT_F16, 8>) : run(launch_forward<CT_F16, 1>);
    }
    return (int)e;
}

// The larger of the two counts of teams that the call may take, by its pointers' alignment.
extern "C" int64_t ct_layer_norm_backward_workspace(int64_t rows, int64_t width, int32_t x_dtype, int32_t weight_grad) {
    if (rows <= 0 || width <= 0 || !weight_grad || !known(x_dtype)) return 0;
    const int64_t a = backward_teams(backward_shape(units_of(width, x_dtype, true), true), rows);
    const int64_t b = backward_teams(backward_shape(units_of(width, x_dtype, false), false), rows);
    return (a > b ? a : b) * 2 * width * (int64_t)sizeof(float);
}

extern "C" int ct_layer_norm_backward(const void *x, int32_t x_dtype, const void *w, int32_t w_dtype, const float *mean,
                                      const float *rstd, const void *dy, void *dx, void *dw, void *dbias, int64_t rows,
                                      int64_t width, void *workspace, int64_t workspace_bytes, hipStream_t stream) {
    if (rows < 0 || rows > 0x7fffffff || width <= 0 || width > 0x7fffffff) return -CT_EINVAL_SHAPE;
    if (!known(x_dtype) || ((w || dw || dbias) && !known(w_dtype))) return -CT_EINVAL_DTYPE;
    if (rows && (!x || !mean || !rstd || !dy)) return -CT_EINVAL_POINTER;
    const bool grad = dw || dbias;
    float *partial = static_cast<float *>(workspace);
    int64_t teams = 0;
    if (rows) {
        if (grad && (!workspace || workspace_bytes < ct_layer_norm_backward_workspace(rows, width, x_dtype, 1) ||
                     reinterpret_cast<uintptr_t>(workspace) % 4))
            return -CT_EINVAL_WORKSPACE;
        if (!grad) partial = nullptr;
        const bool vec = aligned(x) && aligned(dy) && aligned(dx) && aligned(w) && width % (x_dtype == CT_F32 ? 4 : 8) == 0;
        teams = backward_teams(backward_shape(units_of(width, x_dtype, vec), vec), rows);
        const auto run = [&](auto launch) {
            return launch(x, w, w_dtype, mean, rstd, dy, dx, partial, teams, rows, width, stream);
        };
        hipError_t e = hipSuccess;
        if (dx || grad) {
            if (x_dtype == CT_F32) e = vec ? run(launch_backward<CT_F32, 4>) : run(launch_backward<CT_F32, 1>);
            else if (x_dtype == CT_BF16) e = vec ? run(launch_backward<CT_BF16, 8>) : run(launch_backward<CT_BF16, 1>);
            else e = vec ? run(launch_backward<CT_F16, 8>) : run(launch_backward<CT_F16, 1>);
        }
        if (e != hipSuccess) return (int)e;
    }
    if (grad) {
        join_kernel<<<dim3((unsigned)cdiv(width, 64), 2), dim3(1024), 0, stream>>>(partial, teams, width, dw, dbias, w_dtype);
        return (int)hipGetLastError();
    }
    return 0;
}
