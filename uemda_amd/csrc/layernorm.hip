// Layer normalisation over the last (channel) dimension of feature rows, forward and backward.
//   y = (x - mean) * rstd * gamma + beta,   mean = sum x / C,   rstd = 1 / sqrt(sum (x - mean)^2 / C + eps)
//   dx = rstd * (g - mean(g) - xhat * mean(g * xhat)),  g = dy * gamma,  xhat = (x - mean) * rstd
//   dgamma = sum_rows dy * xhat,   dbeta = sum_rows dy
// Bound by HBM: 2 row reads/writes forward, 3 backward, ~8 / ~14 flops an element (32768 x 2048 fp32: 87 us = 6.2 TB/s, 151 = 5.3).  A row is read ONCE: a team of lanes keeps it in
// registers between the two sums of the statistics (the squares are summed about the mean, in 32 bits) and the output, so a row costs
// its bytes and two reductions by lane exchange.  Backward, a team walks rows with its columns fixed, so dgamma / dbeta accumulate in
// registers too; a block's teams are joined in LDS and the blocks' partial sums by a second small launch, in a fixed order: the result
// does not depend on timing.
#include "common.h"

#include <algorithm>

typedef unsigned short bf16_t;

namespace {

template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(const float* p, float* v) {
        const float4 u = *reinterpret_cast<const float4*>(p);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
    static __device__ __forceinline__ void store(float* p, const float* v) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
    static __device__ __forceinline__ float load1(const float* p) { return *p; }
    static __device__ __forceinline__ void store1(float* p, float v) { *p = v; }
};
template <> struct Vec<bf16_t> {
    static constexpr int N = 8;
    static __device__ __forceinline__ unsigned bits(float f) { return (unsigned)__builtin_bit_cast(unsigned short, (__bf16)f); }   // to nearest even: outputs are rounded once
    static __device__ __forceinline__ void load(const bf16_t* p, float* v) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ void store(bf16_t* p, const float* v) {
        *reinterpret_cast<uint4*>(p) = make_uint4(bits(v[0]) | (bits(v[1]) << 16), bits(v[2]) | (bits(v[3]) << 16),
                                                  bits(v[4]) | (bits(v[5]) << 16), bits(v[6]) | (bits(v[7]) << 16));
    }
    static __device__ __forceinline__ float load1(const bf16_t* p) { return __uint_as_float((uint32_t)*p << 16); }
    static __device__ __forceinline__ void store1(bf16_t* p, float v) { *p = (bf16_t)bits(v); }
};

// gamma / beta are kept in 32 bits or bf16 independently of x
__device__ __forceinline__ float param(const void* p, bool is16, int i) {
    return is16 ? __uint_as_float((uint32_t)((const bf16_t*)p)[i] << 16) : ((const float*)p)[i];
}

struct LnP {
    const void* x; const void* dy; const void* gamma; const void* beta;
    void* y;                      // forward: y; backward: dx
    float* mean; float* rstd;     // [rows] each; forward may be null (nothing to save)
    float* part;                  // backward: [blocks][2][C] or null (no parameter gradients)
    void* dgamma; void* dbeta;    // backward: the gradients themselves, written by a launch of one block (either may be null)
    int64_t rows, x_ld, dy_ld;
    int C, period;
    float eps;
    bool p16;
};

// How a row's elements fall to the accesses of its LPR lanes: access q = i * LPR + lane covers the columns q*W - shift ... + W - 1.
//   MODE 0: rows start on 16-byte boundaries, 16-byte accesses, shift 0
//   MODE 1: dense rows of any length: 16-byte accesses on the allocation's own boundaries, shift = the row's start modulo W; the row's
//           first and last access go element by element.  Rows r and r + period start alike: a team walks rows of ONE start (r mod
//           period), so that its columns stay fixed
//   MODE 2: element by element (short rows that are not aligned, where that is faster or the tensor is not dense)
template <typename T, int LPR, int NV, int MODE>
struct Row {
    static constexpr int W = MODE == 2 ? 1 : Vec<T>::N;
    static __device__ __forceinline__ int col(int i, int lane, int shift) { return (i * LPR + lane) * W - (MODE == 1 ? shift : 0); }
    static __device__ __forceinline__ bool whole(int c, int C) { return MODE == 1 ? (c >= 0 && c + W <= C) : c < C; }
    static __device__ __forceinline__ bool inside(int c, int C) { return MODE == 1 ? (c >= 0 && c < C) : true; }   // element of a !whole MODE 1 access
    // `end`: no access may reach past this element of the row (the allocation's last one, seen from the row).  A row's outer accesses
    // hold elements of the neighbouring rows: read whole and masked, so that every lane's row is one load an access; only the very last
    // row of the tensor has to pick its tail's elements one by one
    static __device__ __forceinline__ void load(const T* p, int C, int lane, int shift, bool on, int64_t end, float (*v)[W]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = col(i, lane, shift);
#pragma unroll
            for (int e = 0; e < W; ++e) v[i][e] = 0.f;
            if (MODE == 1) {
                if (on && c < C) {
                    if (c + W <= end) Vec<T>::load(p + c, v[i]);
                    else
#pragma unroll
                        for (int e = 0; e < W; ++e) if (inside(c + e, C)) v[i][e] = Vec<T>::load1(p + c + e);
                }
#pragma unroll
                for (int e = 0; e < W; ++e) v[i][e] = inside(c + e, C) ? v[i][e] : 0.f;
            } else if (on && c < C) {
                if (MODE == 2) v[i][0] = Vec<T>::load1(p + c);
                else Vec<T>::load(p + c, v[i]);
            }
        }
    }
    static __device__ __forceinline__ void store(T* p, int C, int lane, int shift, const float (*v)[W]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = col(i, lane, shift);
            if (whole(c, C)) {
                if (MODE == 2) Vec<T>::store1(p + c, v[i][0]);
                else Vec<T>::store(p + c, v[i]);
            } else if (MODE == 1) {
#pragma unroll
                for (int e = 0; e < W; ++e) if (inside(c + e, C)) Vec<T>::store1(p + c + e, v[i][e]);
            }
        }
    }
    static __device__ __forceinline__ void params(const void* p, bool p16, float other, int C, int lane, int shift, float (*v)[W]) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c0 = col(i, lane, shift);
            if (MODE != 2 && p != nullptr && !p16 && whole(c0, C)) {           // fp32: 16 bytes at a time, on any 4-byte boundary
#pragma unroll
                for (int e = 0; e < W; e += 4) {
                    struct __attribute__((packed, aligned(4))) F4 { float f[4]; };
                    const F4 u = *reinterpret_cast<const F4*>((const float*)p + c0 + e);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[i][e + k] = u.f[k];
                }
                continue;
            }
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const int c = c0 + e;
                v[i][e] = p != nullptr && c >= 0 && c < C ? param(p, p16, c) : other;
            }
        }
    }
};

// Sums of K values over the LPR lanes of a team, in every lane of it; every lane of the block calls it.  Inside a row of 16 lanes by DPP
// (no LDS round trips: exchange with lane ^ 1, ^ 2, then the mirrored half and the mirrored row); a block's four waves through `red`,
// which alternates between two sets of words, so that one barrier a reduction is enough.
template <int LPR, int K>
__device__ __forceinline__ void team_sums(float (&v)[K], float* red, int& flip) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (LPR >= 64) { v[k] = wave_sum_dpp(v[k]); continue; }
        if (LPR >= 2) v[k] += dpp_take0<0xB1, 0xF>(v[k]);
        if (LPR >= 4) v[k] += dpp_take0<0x4E, 0xF>(v[k]);
        if (LPR >= 8) v[k] += dpp_take0<0x141, 0xF>(v[k]);
        if (LPR >= 16) v[k] += dpp_take0<0x140, 0xF>(v[k]);
        if (LPR >= 32) v[k] += __shfl_xor(v[k], 16, 64);
    }
    if (LPR > 64) {
        float* const r = red + flip * 4 * K;
        flip ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) r[(threadIdx.x >> 6) * K + k] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = (r[k] + r[K + k]) + (r[2 * K + k] + r[3 * K + k]);
    }
}

template <typename T, int LPR, int NV, int MODE>
__global__ __launch_bounds__(256) void layernorm_fwd_kernel(const LnP p) {
    using R = Row<T, LPR, NV, MODE>;
    constexpr int W = R::W, TEAMS = 256 / LPR;
    __shared__ float red[8];
    int flip = 0;
    const int lane = threadIdx.x % LPR;
    const int64_t team = (int64_t)blockIdx.x * TEAMS + threadIdx.x / LPR, teams = (int64_t)gridDim.x * TEAMS;
    const int shift = MODE == 1 ? (int)(((team % p.period) * p.C) & (W - 1)) : 0;      // teams % period == 0: all its rows start alike
    const float inv = 1.f / (float)p.C;
    float ga[NV][W], be[NV][W];
    R::params(p.gamma, p.p16, 1.f, p.C, lane, shift, ga);
    R::params(p.beta, p.p16, 0.f, p.C, lane, shift, be);
    // the loop's bound is uniform over the block: every lane joins every exchange
    for (int64_t base = (int64_t)blockIdx.x * TEAMS, r = team; base < p.rows; base += teams, r += teams) {
        const bool on = r < p.rows;
        float v[NV][W], s[1] = {0.f};
        R::load((const T*)p.x + r * p.x_ld, p.C, lane, shift, on, (p.rows - r) * p.x_ld, v);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < W; ++e) s[0] += v[i][e];
        team_sums<LPR, 1>(s, red, flip);
        const float mean = s[0] * inv;
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = R::col(i, lane, shift);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                v[i][e] -= mean;
                const bool in = MODE == 1 ? R::inside(c + e, p.C) : c < p.C;
                s[0] = in ? fmaf(v[i][e], v[i][e], s[0]) : s[0];
            }
        }
        team_sums<LPR, 1>(s, red, flip);
        const float rstd = 1.f / sqrtf(s[0] * inv + p.eps);
        if (!on) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < W; ++e) v[i][e] = fmaf(v[i][e] * rstd, ga[i][e], be[i][e]);
        R::store((T*)p.y + r * p.C, p.C, lane, shift, v);
        if (p.mean != nullptr && lane == 0) { p.mean[r] = mean; p.rstd[r] = rstd; }
    }
}

// U rows of a team are in flight together: their loads are issued before the first reduction
template <typename T, int LPR, int NV, int MODE, int U>
__global__ __launch_bounds__(256) void layernorm_bwd_kernel(const LnP p) {
    // where column c's sums of this block go
    auto leave = [&](int c, float w, float b) {
        if (gridDim.x > 1) {
            float* const out = p.part + (int64_t)blockIdx.x * 2 * p.C;
            out[c] = w;
            out[p.C + c] = b;
            return;
        }
        auto one = [&](void* to, float v) {
            if (to == nullptr) return;
            if (p.p16) Vec<bf16_t>::store1((bf16_t*)to + c, v);
            else ((float*)to)[c] = v;
        };
        one(p.dgamma, w);
        one(p.dbeta, b);
    };
    using R = Row<T, LPR, NV, MODE>;
    constexpr int W = R::W, TEAMS = 256 / LPR, CAP = LPR > 64 ? 1 : LPR * NV * W;
    __shared__ float red[16 * U];
    __shared__ float join[2][CAP];
    int flip = 0;
    const int lane = threadIdx.x % LPR;
    const int64_t teams = (int64_t)gridDim.x * TEAMS;
    int64_t team = (int64_t)blockIdx.x * TEAMS + threadIdx.x / LPR, block0 = (int64_t)blockIdx.x * TEAMS;      // first row of the team, of the block
    if (MODE == 1 && LPR < 64) {                                               // the teams of a wave on rows that start alike: they add up their columns
        const int w = blockIdx.x * 4 + (threadIdx.x >> 6), w0 = blockIdx.x * 4, per = p.period * (64 / LPR);
        team = (int64_t)(w / p.period) * per + (threadIdx.x & 63) / LPR * p.period + w % p.period;
        block0 = (int64_t)(w0 / p.period) * per + w0 % p.period;
    }
    const int shift = MODE == 1 ? (int)(((team % p.period) * p.C) & (W - 1)) : 0;
    const float inv = 1.f / (float)p.C;
    float ga[NV][W], aw[NV][W], ab[NV][W];
    R::params(p.gamma, p.p16, 1.f, p.C, lane, shift, ga);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < W; ++e) aw[i][e] = ab[i][e] = 0.f;
    for (int64_t base = block0, r = team; base < p.rows; base += teams * U, r += teams * U) {
        float v[U][NV][W], g[U][NV][W], mean[U], rstd[U], s[2 * U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t ru = r + u * teams;
            const bool on = ru < p.rows;
            R::load((const T*)p.x + ru * p.x_ld, p.C, lane, shift, on, (p.rows - ru) * p.x_ld, v[u]);
            R::load((const T*)p.dy + ru * p.dy_ld, p.C, lane, shift, on, (p.rows - ru) * p.dy_ld, g[u]);
            mean[u] = on ? p.mean[ru] : 0.f;
            rstd[u] = on ? p.rstd[ru] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const float h = (v[u][i][e] - mean[u]) * rstd[u];          // columns outside the row carry dy = 0
                    v[u][i][e] = h;
                    aw[i][e] = fmaf(g[u][i][e], h, aw[i][e]);
                    ab[i][e] += g[u][i][e];
                    g[u][i][e] *= ga[i][e];
                    s1 += g[u][i][e];
                    s2 = fmaf(g[u][i][e], h, s2);
                }
            s[2 * u] = s1;
            s[2 * u + 1] = s2;
        }
        team_sums<LPR, 2 * U>(s, red, flip);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t ru = r + u * teams;
            if (ru >= p.rows) continue;
            const float s1 = s[2 * u] * inv, s2 = s[2 * u + 1] * inv;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < W; ++e) v[u][i][e] = rstd[u] * (g[u][i][e] - s1 - v[u][i][e] * s2);
            R::store((T*)p.y + ru * p.C, p.C, lane, shift, v[u]);
        }
    }
    if (p.part == nullptr) return;
    if (LPR > 64) {                                                            // one team a block: straight out
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const int c = R::col(i, lane, shift) + e;
                if (c >= 0 && c < p.C) leave(c, aw[i][e], ab[i][e]);
            }
        return;
    }
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1)                                         // the teams of a wave
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < W; ++e) { aw[i][e] += __shfl_xor(aw[i][e], o, 64); ab[i][e] += __shfl_xor(ab[i][e], o, 64); }
    for (int w = 0; w < 4; ++w) {                                              // the waves, in order
        if ((int)(threadIdx.x >> 6) == w && (threadIdx.x & 63) < LPR) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const int c = R::col(i, lane, shift) + e;
                    if (c >= 0 && c < p.C) {
                        join[0][c] = aw[i][e] + (w ? join[0][c] : 0.f);
                        join[1][c] = ab[i][e] + (w ? join[1][c] : 0.f);
                    }
                }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < p.C; c += 256) leave(c, join[0][c], join[1][c]);
}

// Any row length, any alignment: a block per row that reads the row again for each sum (rows beyond the register kernels' 8192
// columns, or rows whose strides and bases share no 16-byte grid).  The parameter gradients are a separate pass over columns.
// A thread's share has no bound here, so where it is long (A: double) these sums are kept in 64 bits: in 32, the mean of 2^24 elements around 100
// was off by 0.05, five times their deviation.  A share of up to 32 elements of a row is as good in 32 bits, and the reductions are shorter: 65536 x
// 513 bf16 that begin anywhere 102 us forward and 175 backward, so 126 and 203 in 64; 4096 x 20001 184 and 320, so 188 and 324.
template <typename A> __device__ __forceinline__ A block_sum(A v, A* red) {
    if constexpr (sizeof(A) == 8) v = wave_sum_d(v);
    else v = wave_sum_dpp(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}
__device__ __forceinline__ float mul_add(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double mul_add(double a, double b, double c) { return fma(a, b, c); }
template <typename T, typename A>
__global__ __launch_bounds__(256) void layernorm_fwd_any_kernel(const LnP p) {
    __shared__ A red[4];
    const A inv = A(1) / (A)p.C;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* const x = (const T*)p.x + r * p.x_ld;
        T* const y = (T*)p.y + r * p.C;
        A s = 0, q = 0;
        for (int c = threadIdx.x; c < p.C; c += 256) s += (A)Vec<T>::load1(x + c);
        const float mean = (float)(block_sum<A>(s, red) * inv);
        for (int c = threadIdx.x; c < p.C; c += 256) { const A d = (A)(Vec<T>::load1(x + c) - mean); q = mul_add(d, d, q); }
        const float rstd = 1.f / sqrtf((float)(block_sum<A>(q, red) * inv) + p.eps);
        for (int c = threadIdx.x; c < p.C; c += 256) {
            const float ga = p.gamma ? param(p.gamma, p.p16, c) : 1.f, be = p.beta ? param(p.beta, p.p16, c) : 0.f;
            Vec<T>::store1(y + c, fmaf((Vec<T>::load1(x + c) - mean) * rstd, ga, be));
        }
        if (p.mean != nullptr && threadIdx.x == 0) { p.mean[r] = mean; p.rstd[r] = rstd; }
    }
}
template <typename T, typename A>
__global__ __launch_bounds__(256) void layernorm_bwd_any_kernel(const LnP p) {
    __shared__ A red[4];
    const A inv = A(1) / (A)p.C;
    for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const T* const x = (const T*)p.x + r * p.x_ld;
        const T* const dy = (const T*)p.dy + r * p.dy_ld;
        T* const dx = (T*)p.y + r * p.C;
        const float mean = p.mean[r], rstd = p.rstd[r];
        A t1 = 0, t2 = 0;
        for (int c = threadIdx.x; c < p.C; c += 256) {
            const float g = Vec<T>::load1(dy + c) * (p.gamma ? param(p.gamma, p.p16, c) : 1.f);
            t1 += (A)g;
            t2 = mul_add((A)g, (A)((Vec<T>::load1(x + c) - mean) * rstd), t2);
        }
        const float s1 = (float)(block_sum<A>(t1, red) * inv), s2 = (float)(block_sum<A>(t2, red) * inv);
        for (int c = threadIdx.x; c < p.C; c += 256) {
            const float g = Vec<T>::load1(dy + c) * (p.gamma ? param(p.gamma, p.p16, c) : 1.f);
            Vec<T>::store1(dx + c, rstd * (g - s1 - (Vec<T>::load1(x + c) - mean) * rstd * s2));
        }
    }
}
// 64 columns x 4 row lanes a block, rows shared out over gridDim.y
template <typename T, typename A>
__global__ __launch_bounds__(256) void layernorm_cols_kernel(const LnP p) {
    __shared__ A join[2][4][64];
    const int w = threadIdx.x >> 6;
    for (int64_t c0 = (int64_t)blockIdx.x * 64; c0 < p.C; c0 += (int64_t)gridDim.x * 64) {
        const int64_t c = c0 + (threadIdx.x & 63);
        A a = 0, b = 0;
        if (c < p.C)
            for (int64_t r = (int64_t)blockIdx.y * 4 + w; r < p.rows; r += (int64_t)gridDim.y * 4) {
                const float g = Vec<T>::load1((const T*)p.dy + r * p.dy_ld + c);
                a = mul_add((A)g, (A)((Vec<T>::load1((const T*)p.x + r * p.x_ld + c) - p.mean[r]) * p.rstd[r]), a);
                b += (A)g;
            }
        join[0][w][threadIdx.x & 63] = a;
        join[1][w][threadIdx.x & 63] = b;
        __syncthreads();
        if (w < 2 && c < p.C) {
            const A* const j = &join[w][0][threadIdx.x & 63];
            p.part[((int64_t)blockIdx.y * 2 + w) * p.C + c] = (float)((j[0] + j[64]) + (j[128] + j[192]));
        }
        __syncthreads();
    }
}

// dgamma / dbeta = the blocks' partial sums, added in a fixed order: 16 columns x 64 slices of the blocks a block of 1024 threads
__global__ __launch_bounds__(1024) void layernorm_params_kernel(const float* __restrict__ part, int nb, int C, void* dgamma, void* dbeta, bool p16) {
    __shared__ float join[64][17];
    const int t = threadIdx.x & 15, sl = threadIdx.x >> 4;
    const int64_t n = 2 * (int64_t)C;
    for (int64_t c0 = (int64_t)blockIdx.x * 16; c0 < n; c0 += (int64_t)gridDim.x * 16) {
        const int64_t col = c0 + t;
        float s = 0.f;
        if (col < n) {
#pragma unroll 8
            for (int b = sl; b < nb; b += 64) s += part[b * n + col];
        }
        join[sl][t] = s;
        __syncthreads();
        if (sl < 4) {
            float q = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) q += join[sl * 16 + i][t];
            q += __shfl_xor(q, 16, 64);
            q += __shfl_xor(q, 32, 64);
            void* const out = col < C ? dgamma : dbeta;
            const int64_t c = col < C ? col : col - C;
            if (sl == 0 && col < n && out != nullptr) {
                if (p16) Vec<bf16_t>::store1((bf16_t*)out + c, q);
                else ((float*)out)[c] = q;
            }
        }
        __syncthreads();
    }
}

// most blocks the backward of so many rows takes: each leaves its partial sums, which are to stay a fraction of what its rows read and write
// (2000 x 2048 bf16: 256 blocks 19 us, 768 22, 1536 33)
int64_t bwd_blocks(int64_t rows) {
    const int64_t n = uem_cdiv(rows < 256 ? rows : rows < 2048 ? 256 : rows / 8, 8) * 8;
    return n > 2048 ? 2048 : n;
}
// a launch has fewer than 2^32 threads in a dimension: rows of more columns than so many blocks cover are walked in turns
constexpr int64_t MOST_BLOCKS = 1 << 20;
// blocks of a kernel that a CU holds at once (registers): asked for once
template <typename K> int resident(K kernel) {
    int n = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 256, 0) != hipSuccess || n < 1) n = 4;
    return n > 8 ? 8 : n;
}

template <typename T, int LPR, int NV, int MODE>
int go(const LnP& p, bool bwd, hipStream_t st) {
    // Grids that the chip holds at once: another block of a CU's would run behind the others, and where rows cost instructions (bf16, or rows
    // that are not aligned) fewer leave them uncovered.  Measured, us (2^26 elements unless said), backward, 512 / 768 / 1024 / 1536 / 2048 blocks:
    //   bf16 of 2^27: 256 columns (4 a CU) 233 / 177 / 152 / 186 / 159, 2048 (6) 267 / 207 / 177 / 162 / 199; bf16 777 (3) 165 / 126 / 176 / 136 / 153,
    //   33 (8) 1252 / 854 / 657 / 469 / 374; fp32 1001 204 / 155 / 163 / 175 / 179.
    // Aligned fp32 rows are so few instructions a byte that two blocks a CU, three where a lane holds one access, do best: 2^27 elements
    //   in 256 columns 290 / 293 / 301 / 323 / 330, 2048 289 / 294 / 323 / 326 / 324, 1024 312 / 287 / 296 / 324 / 324.
    // forward, 1024 / 1536 / 2048 / 16384: bf16 2049 columns (6) 81 / 65 / 82 / 104, 4096 (6) 52 / 44 / 53 / 61; fp32 7 (8) 276 / 218 / 190 / 194.
    //   Aligned rows of up to a wave, and fp32 ones, are fastest with a block for as few rows as there are: 256 columns bf16 48 / 46 / 46 / 44,
    //   fp32 98 / 103 / 110 / 98 (91 with 65536 blocks).
    // Two rows in flight a team gain where a team is part of a wave, backward alone: 168 against 157.
    constexpr int UB = LPR < 64 ? 2 : 1, TEAMS = 256 / LPR;
    constexpr bool f32 = sizeof(T) == 4;
    auto grid = [&](int rows, int64_t most) {
        int64_t n = uem_cdiv(p.rows, rows);
        if (n > most) n = most;
        return (int)(MODE == 1 ? uem_cdiv(n, 8) * 8 : n);                      // teams % period == 0 (period <= 8)
    };
    if (!bwd) {
        static const int fit = resident(layernorm_fwd_kernel<T, LPR, NV, MODE>);
        const int nb = grid(TEAMS, MODE == 0 && (f32 || LPR <= 64) ? 16384 : 256 * fit);
        layernorm_fwd_kernel<T, LPR, NV, MODE><<<nb, 256, 0, st>>>(p);
        return nb;
    }
    if constexpr (!(f32 && MODE == 1 && LPR < 64)) {                           // (such rows go forward only: run)
        static const int fit = resident(layernorm_bwd_kernel<T, LPR, NV, MODE, UB>);
        const int few = MODE == 1 || (LPR > 64 && NV == 1) ? 3 : 2;
        const int64_t most = 256 * (f32 && MODE != 2 && fit > few ? few : fit), leave = bwd_blocks(p.rows);
        const int nb = grid(TEAMS * UB, most < leave ? most : leave);
        layernorm_bwd_kernel<T, LPR, NV, MODE, UB><<<nb, 256, 0, st>>>(p);
        return nb == 1 ? 0 : nb;                                               // 0: no partial sums left
    }
    return 0;
}

// dense rows of C elements r and r + period start alike modulo w elements
int period_of(int C, int w) {
    int n = w;
    while (n > 1 && ((int64_t)(n / 2) * C) % w == 0) n /= 2;
    return n;
}
template <typename T>
int run(LnP p, bool bwd, hipStream_t st) {
    constexpr int W = Vec<T>::N;
    const uintptr_t bases = (uintptr_t)p.x | (uintptr_t)p.y | (bwd ? (uintptr_t)p.dy : 0);
    const bool base16 = (bases & 15) == 0;
    const bool dense = p.x_ld == p.C && (!bwd || p.dy_ld == p.C);
    p.period = 1;
    // Lanes per row: as many as it has accesses; one wave while a lane holds at most 16 elements (8 in bf16's wide accesses), a block of four above -- backward keeps
    // five values an element in registers (x, g, gamma and the two parameter gradients), 32 elements a lane would leave two waves a SIMD
    if (base16 && p.C % W == 0 && p.x_ld % W == 0 && (!bwd || p.dy_ld % W == 0)) {
        const int v = p.C / W;
        if (v <= 1) return go<T, 1, 1, 0>(p, bwd, st);
        if (v <= 2) return go<T, 2, 1, 0>(p, bwd, st);
        if (v <= 4) return go<T, 4, 1, 0>(p, bwd, st);
        if (v <= 8) return go<T, 8, 1, 0>(p, bwd, st);
        if (v <= 16) return go<T, 16, 1, 0>(p, bwd, st);
        if (v <= 32) return go<T, 32, 1, 0>(p, bwd, st);
        if (v <= 64) return go<T, 64, 1, 0>(p, bwd, st);
        if (v <= 128) return go<T, 64, 2, 0>(p, bwd, st);
        if (v <= 256) return go<T, 256, 1, 0>(p, bwd, st);
        if (v <= 512) return go<T, 256, 2, 0>(p, bwd, st);
        if (v <= 1024) return go<T, 256, 4, 0>(p, bwd, st);
        if (W == 4 && v <= 2048) return go<T, 256, W == 4 ? 8 : 4, 0>(p, bwd, st);
    } else if (base16 && dense && p.C > 8 && (W == 8 ? p.C <= 256 : !bwd && p.C <= 64)) {
        // Short rows in whole accesses, against element by element, us at 2^26 elements: bf16 forward 33 columns 273 / 129, 100 158 / 80, 255 133 / 93,
        // backward 33 379 / 221, 100 225 / 130, 255 170 / 128; at 2^25 forward 7 82 / 78, backward 7 110 / 214, 9 298 / 212, 13 214 / 157.  fp32, twice the
        // bytes an element: forward 33 278 / 195, 67 170 / 169, 131 130 / 156; backward 33 249 / 277, 131 186 / 221, at 2^25 9 172 / 227.
        const int v = (p.C + W - 1 + W - 1) / W;                               // accesses of the worst start
        p.period = period_of(p.C, W);
        if (v <= 2) return go<T, 2, 1, 1>(p, bwd, st);
        if (v <= 4) return go<T, 4, 1, 1>(p, bwd, st);
        if (v <= 8) return go<T, 8, 1, 1>(p, bwd, st);
        if (v <= 16) return go<T, 16, 1, 1>(p, bwd, st);
        if (v <= 32) return go<T, 32, 1, 1>(p, bwd, st);
        if (W == 8) return go<T, 64, W == 8 ? 1 : 2, 1>(p, bwd, st);
    } else if (p.C <= 256) {
        if (p.C <= 4) return go<T, 4, 1, 2>(p, bwd, st);
        if (p.C <= 8) return go<T, 8, 1, 2>(p, bwd, st);
        if (p.C <= 32) return go<T, 32, 1, 2>(p, bwd, st);
        if (p.C <= 64) return go<T, 64, 1, 2>(p, bwd, st);
        return go<T, 64, 4, 2>(p, bwd, st);
    } else if (base16 && dense) {
        const int v = (p.C + W - 1 + W - 1) / W;                               // accesses of the worst start
        p.period = period_of(p.C, W);
        if (v <= 128) return go<T, 64, 2, 1>(p, bwd, st);
        if (v <= 256) return go<T, 256, 1, 1>(p, bwd, st);
        if (v <= 512) return go<T, 256, 2, 1>(p, bwd, st);
        if (v <= 1024) return go<T, 256, 4, 1>(p, bwd, st);
        if (W == 4 && v <= 2048) return go<T, 256, W == 4 ? 8 : 4, 1>(p, bwd, st);
    }
    const int nb = p.rows < 256 * 16 ? (int)p.rows : 256 * 16;
    const bool far = p.C > 8192;
    if (!bwd) {
        if (far) layernorm_fwd_any_kernel<T, double><<<nb, 256, 0, st>>>(p);
        else layernorm_fwd_any_kernel<T, float><<<nb, 256, 0, st>>>(p);
        return nb;
    }
    if (far) layernorm_bwd_any_kernel<T, double><<<nb, 256, 0, st>>>(p);
    else layernorm_bwd_any_kernel<T, float><<<nb, 256, 0, st>>>(p);
    if (p.part == nullptr) return nb;
    const int ny = (int)(uem_cdiv(p.rows, 4) < 64 ? uem_cdiv(p.rows, 4) : 64);
    const dim3 grid((unsigned)std::min<int64_t>(uem_cdiv(p.C, 64), MOST_BLOCKS), (unsigned)ny);
    if (p.rows > 65536) layernorm_cols_kernel<T, double><<<grid, 256, 0, st>>>(p);       // a thread's share: rows / 256
    else layernorm_cols_kernel<T, float><<<grid, 256, 0, st>>>(p);
    return ny;
}

}  // namespace

extern "C" int64_t uem_layernorm_workspace_floats(int64_t rows, int C) {
    int64_t n = bwd_blocks(rows);
    if (C > 8192 && n > 64) n = 64;                                            // longer rows: the pass over columns
    return n * 2 * (int64_t)C;
}
extern "C" int uem_layernorm_fwd(const void* x, int64_t x_ld, const void* gamma, const void* beta, void* y, float* mean, float* rstd,
                                 int64_t rows, int C, float eps, int flags, void* stream) {
    UEM_REQUIRE(x && y && rows > 0 && C > 0 && C <= (1 << 30) && x_ld >= C, "layernorm_fwd: bad arguments (rows > 0, 0 < C <= 2^30, x_ld >= C)");
    UEM_REQUIRE((mean == nullptr) == (rstd == nullptr), "layernorm_fwd: mean and rstd go together");
    UEM_REQUIRE((flags & ~(UEM_LN_BF16 | UEM_LN_PARAM_BF16)) == 0, "layernorm_fwd: unknown flags %d", flags);
    LnP p{};
    p.x = x; p.gamma = gamma; p.beta = beta; p.y = y; p.mean = mean; p.rstd = rstd; p.rows = rows; p.x_ld = x_ld; p.C = C; p.eps = eps;
    p.p16 = (flags & UEM_LN_PARAM_BF16) != 0;
    if (flags & UEM_LN_BF16) run<bf16_t>(p, false, (hipStream_t)stream);
    else run<float>(p, false, (hipStream_t)stream);
    return uem_check_launch("layernorm_fwd");
}
extern "C" int uem_layernorm_bwd(const void* x, int64_t x_ld, const void* dy, int64_t dy_ld, const void* gamma, const float* mean,
                                 const float* rstd, void* dx, void* dgamma, void* dbeta, float* workspace, int64_t rows, int C, int flags,
                                 void* stream) {
    UEM_REQUIRE(x && dy && mean && rstd && dx && rows > 0 && C > 0 && C <= (1 << 30) && x_ld >= C && dy_ld >= C,
                "layernorm_bwd: bad arguments (rows > 0, 0 < C <= 2^30, strides >= C)");
    UEM_REQUIRE((dgamma == nullptr && dbeta == nullptr) || workspace, "layernorm_bwd: parameter gradients need the workspace");
    UEM_REQUIRE((flags & ~(UEM_LN_BF16 | UEM_LN_PARAM_BF16)) == 0, "layernorm_bwd: unknown flags %d", flags);
    LnP p{};
    p.x = x; p.dy = dy; p.gamma = gamma; p.y = dx; p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
    p.part = dgamma || dbeta ? workspace : nullptr;
    p.dgamma = dgamma; p.dbeta = dbeta;
    p.rows = rows; p.x_ld = x_ld; p.dy_ld = dy_ld; p.C = C; p.p16 = (flags & UEM_LN_PARAM_BF16) != 0;
    hipStream_t st = (hipStream_t)stream;
    const int nb = (flags & UEM_LN_BF16) ? run<bf16_t>(p, true, st) : run<float>(p, true, st);
    if (p.part && nb > 0) layernorm_params_kernel<<<(int)std::min<int64_t>(uem_cdiv(2 * (int64_t)C, 16), MOST_BLOCKS), 1024, 0, st>>>(p.part, nb, C, dgamma, dbeta, p.p16);
    return uem_check_launch("layernorm_bwd");
}
