// clip_grad_norm_(max_norm, L2) + SGD(momentum, weight_decay) fused over the flat parameter arena.
// Reference: tools/train_ssl_uem.py:169-170,228-232 (torch.optim.SGD + clip_grad.clip_grad_norm_).
#include "common.h"

__global__ __launch_bounds__(256) void sqnorm_partial_kernel(const float* __restrict__ g, int64_t n, float* __restrict__ partial) {
    double s = 0.0;
    const int64_t nvec = n >> 2;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nvec; i += (int64_t)gridDim.x * 256) {
        const float4 v = reinterpret_cast<const float4*>(g)[i];
        s += (double)v.x * v.x + (double)v.y * v.y + (double)v.z * v.z + (double)v.w * v.w;
    }
    if (blockIdx.x == 0)
        for (int64_t i = (nvec << 2) + threadIdx.x; i < n; i += 256) s += (double)g[i] * g[i];
    __shared__ double red[4];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) partial[blockIdx.x] = (float)((red[0] + red[1]) + (red[2] + red[3]));
}
__global__ __launch_bounds__(256) void sqnorm_final_kernel(const float* __restrict__ partial, int nb, float* __restrict__ out) {
    double s = 0.0;
    for (int i = threadIdx.x; i < nb; i += 256) s += partial[i];
    __shared__ double red[4];
    s = wave_sum_d(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) out[0] = (float)sqrt((red[0] + red[1]) + (red[2] + red[3]));
}
extern "C" int uem_grad_sqnorm(const float* grad, int64_t n, float* partial, float* norm_out, void* stream) {
    UEM_REQUIRE(grad && partial && norm_out && n > 0, "grad_sqnorm: bad arguments");
    UEM_REQUIRE(((uintptr_t)grad & 15) == 0, "grad_sqnorm: grad must be 16-byte aligned");
    hipStream_t st = (hipStream_t)stream;
    int nb = (int)uem_cdiv(n / 4 + 1, 256 * 4);
    if (nb > UEM_NORM_BLOCKS) nb = UEM_NORM_BLOCKS;
    sqnorm_partial_kernel<<<nb, 256, 0, st>>>(grad, n, partial);
    sqnorm_final_kernel<<<1, 256, 0, st>>>(partial, nb, norm_out);
    return uem_check_launch("grad_sqnorm");
}

__global__ __launch_bounds__(256) void sgd_clip_kernel(float* __restrict__ p, float* __restrict__ g, float* __restrict__ buf,
                                                       int64_t n, const float* __restrict__ norm, float max_norm, float lr,
                                                       float momentum, float wd, int first, float prescale,
                                                       const float* __restrict__ lr_dev) {
    // lr_dev (optional): the learning rate as a DEVICE scalar -- a step captured in a hipGraph bakes by-value arguments in, the
    // schedule then writes this word before every replay
    if (lr_dev) lr = lr_dev[0];
    // clip coefficient exactly as torch.nn.utils.clip_grad_norm_: min(max_norm / (total_norm + 1e-6), 1)
    float coef = 1.0f;
    if (norm) { coef = max_norm / (norm[0] * prescale + 1e-6f); coef = coef > 1.0f ? 1.0f : coef; }
    coef *= prescale;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const float gi = g[i] * coef;
        g[i] = gi;                                        // clip_grad_norm_ scales .grad in place
        const float d = gi + wd * p[i];
        const float b = first ? d : momentum * buf[i] + d;
        buf[i] = b;
        p[i] = p[i] - lr * b;
    }
}
extern "C" int uem_sgd_clip_step(float* param, float* grad, float* momentum_buf, int64_t n, const float* norm, float max_norm,
                                 float lr, float momentum, float weight_decay, int first_step, float grad_prescale,
                                 const float* lr_dev, void* stream) {
    UEM_REQUIRE(param && grad && momentum_buf && n > 0, "sgd_clip_step: bad arguments");
    sgd_clip_kernel<<<uem_stream_grid(n, 256), 256, 0, (hipStream_t)stream>>>(param, grad, momentum_buf, n, norm, max_norm, lr,
                                                                             momentum, weight_decay, first_step, grad_prescale, lr_dev);
    return uem_check_launch("sgd_clip_step");
}

// ---- the global norm over MANY tensors, and clipping ---------------------------------------------------------------------------------
// n = sqrt(sum over all tensors of g^2) (or max |g|), then g *= min(max_norm / (n + 1e-6), 1) in place.
// Bound by HBM: one read for the norm, one read and one write where something is clipped (the second read comes out of the 256 MB last-level
// cache as far as the list fits: the scaling pass walks the list backwards).  The tensors are named to the kernels BY VALUE, up to MT_MOST a
// launch: no table in device memory, nothing to keep alive, and a captured launch carries its own list.  A block takes one run of 16-byte
// accesses of one tensor; a tensor may begin and end anywhere, its outer elements are taken one by one.  Squares are exact in 64 bits for
// both types and summed there (no overflow at 1e20, no loss over 10^9 elements).  The partial sums are added in one order and without
// atomics: by every block of the scaling pass itself while they are few (one launch less), by a block of their own beyond MT_JOIN.
// Measured, 400 M elements in 600 tensors (1.0 GB, half the tensors bf16): 2048 blocks 240 + 457 us (norm, scaling), 8192 blocks
// 180 + 365 us = 5.5 TB/s either way, what a copy moves; 175 tensors of a ResNet-50 with heads (98 MB): 21 + 31 us.
typedef unsigned short bf16_t;
constexpr int MT_MOST = 216;                      // tensors a launch: 3.9 KB of the 4 KB of kernel arguments
constexpr int MT_JOIN = 1024;                     // up to so many partial sums are added up by every block of the scaling pass itself
constexpr int MT_BLOCKS = UEM_MULTI_BLOCKS;       // blocks the whole list is cut into, beside one or two more per tensor (its outer accesses)
struct MtList {
    void* ptr[MT_MOST];
    int64_t n[MT_MOST];
    uint16_t start[MT_MOST + 1];                  // first block of each tensor in this launch
    unsigned bf16[(MT_MOST + 31) / 32];
    int count, part0, run;                        // tensors; first partial sum; 16-byte accesses a block
};
struct MtRun {                                    // what one block does
    char* base;                                   // of access 0, on a 16-byte boundary
    int64_t lo, hi, first, last;                  // accesses [lo, hi); elements [first, last) counted from base
    bool is16;
};
__device__ __forceinline__ MtRun mt_run(const MtList& l, int b) {
    int t = 0;
    static_assert(MT_MOST <= 256 && sizeof(MtList) <= 4000, "a launch's list");
    for (int step = 128; step > 0; step >>= 1)    // last tensor that starts at or before block b
        if (t + step < l.count && l.start[t + step] <= b) t += step;
    MtRun r;
    r.is16 = (l.bf16[t >> 5] >> (t & 31)) & 1;
    const uintptr_t p = (uintptr_t)l.ptr[t];
    r.base = (char*)(p & ~(uintptr_t)15);
    const int size = r.is16 ? 2 : 4, per = 16 / size;
    r.first = (int64_t)(p & 15) / size;
    r.last = r.first + l.n[t];
    r.lo = (int64_t)(b - l.start[t]) * l.run;
    const int64_t end = (r.last + per - 1) / per;
    r.hi = r.lo + l.run < end ? r.lo + l.run : end;
    return r;
}
template <bool IS16>
__device__ __forceinline__ float mt_elem(const char* base, int64_t i) {
    return IS16 ? __uint_as_float((uint32_t)((const bf16_t*)base)[i] << 16) : ((const float*)base)[i];
}
template <bool IS16>
__device__ __forceinline__ void mt_unpack(const uint4 u, float* v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (IS16) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        else v[i] = __uint_as_float(w[i]);
    }
}
// one step of the reduction: L2 adds the square; MAX keeps the largest magnitude as its bit pattern (a NaN's lies above infinity's)
template <bool MAX>
__device__ __forceinline__ void mt_take(double& s, uint32_t& m, float v) {
    if (MAX) { const uint32_t u = __float_as_uint(v) & 0x7fffffffu; m = u > m ? u : m; }
    else s = fma((double)v, (double)v, s);
}
template <bool IS16, bool MAX>
__device__ __forceinline__ void mt_reduce(const MtRun& r, double& s, uint32_t& m) {
    constexpr int PER = IS16 ? 8 : 4;
    // whole accesses: all of [lo, hi) but a tensor's outer ones
    const int64_t wlo = r.lo == 0 && r.first > 0 ? 1 : r.lo, whi = r.hi * PER > r.last ? r.hi - 1 : r.hi;
    int64_t i = wlo + threadIdx.x;
    double s2 = 0.0;
    for (; i + 3 * 256 < whi; i += 4 * 256) {
        uint4 u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = ((const uint4*)r.base)[i + k * 256];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float v[PER];
            mt_unpack<IS16>(u[k], v);
#pragma unroll
            for (int e = 0; e < PER; ++e) mt_take<MAX>((e & 1) ? s2 : s, m, v[e]);
        }
    }
    for (; i < whi; i += 256) {
        float v[PER];
        mt_unpack<IS16>(((const uint4*)r.base)[i], v);
#pragma unroll
        for (int e = 0; e < PER; ++e) mt_take<MAX>((e & 1) ? s2 : s, m, v[e]);
    }
    s += s2;
    // the outer accesses, element by element: at most PER - 1 elements on either side (both sides are one access in a tiny tensor)
    if (threadIdx.x < PER && wlo > r.lo) {
        const int64_t e = threadIdx.x;
        if (e >= r.first && e < r.last) mt_take<MAX>(s, m, mt_elem<IS16>(r.base, e));
    }
    if (threadIdx.x < PER && whi < r.hi && whi >= wlo) {
        const int64_t e = whi * PER + threadIdx.x;
        if (e < r.last) mt_take<MAX>(s, m, mt_elem<IS16>(r.base, e));
    }
}
template <bool MAX>
__global__ __launch_bounds__(256) void multi_norm_partial_kernel(const MtList l, double* __restrict__ partial) {
    const MtRun r = mt_run(l, blockIdx.x);
    double s = 0.0;
    uint32_t m = 0;
    if (r.is16) mt_reduce<true, MAX>(r, s, m);
    else mt_reduce<false, MAX>(r, s, m);
    __shared__ double red[4];
    if (MAX) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) { const uint32_t u = __shfl_xor(m, o, 64); m = u > m ? u : m; }
        s = __hiloint2double(0, (int)m);
    } else {
        s = wave_sum_d(s);
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        if (MAX) {
            for (int i = 1; i < 4; ++i) { const uint32_t u = (uint32_t)__double2loint(red[i]); m = u > m ? u : m; }
            partial[l.part0 + blockIdx.x] = __hiloint2double(0, (int)m);
        } else {
            partial[l.part0 + blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
        }
    }
}
// the norm from all partial sums: the same value in every thread of every block that calls it
template <bool MAX, int NT>
__device__ __forceinline__ float mt_norm(const double* __restrict__ partial, int np) {
    __shared__ double red[NT / 64];
    double s = 0.0;
    uint32_t m = 0;
    for (int i = threadIdx.x; i < np; i += NT) {
        if (MAX) { const uint32_t u = (uint32_t)__double2loint(partial[i]); m = u > m ? u : m; }
        else s += partial[i];
    }
    if (MAX) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) { const uint32_t u = __shfl_xor(m, o, 64); m = u > m ? u : m; }
        s = __hiloint2double(0, (int)m);
    } else {
        s = wave_sum_d(s);
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
    m = 0;
    for (int i = 0; i < NT / 64; ++i) {
        const uint32_t u = (uint32_t)__double2loint(red[i]);
        s += red[i];
        m = u > m ? u : m;
    }
    return MAX ? __uint_as_float(m) : (float)sqrt(s);
}
template <bool MAX>
__global__ __launch_bounds__(1024) void multi_norm_final_kernel(const double* __restrict__ partial, int np, float* __restrict__ out) {
    const float n = mt_norm<MAX, 1024>(partial, np);
    if (threadIdx.x == 0) out[0] = n;
}
template <bool IS16>
__device__ __forceinline__ void mt_scale(const MtRun& r, float coef) {
    constexpr int PER = IS16 ? 8 : 4;
    const int64_t wlo = r.lo == 0 && r.first > 0 ? 1 : r.lo, whi = r.hi * PER > r.last ? r.hi - 1 : r.hi;
    auto scaled = [&](const uint4 u) {
        float v[PER];
        mt_unpack<IS16>(u, v);
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (IS16)                              // the product in 32 bits, rounded once, to nearest even
                w[k] = (uint32_t)__builtin_bit_cast(unsigned short, (__bf16)(v[2 * k] * coef)) |
                       ((uint32_t)__builtin_bit_cast(unsigned short, (__bf16)(v[2 * k + 1] * coef)) << 16);
            else w[k] = __float_as_uint(v[k] * coef);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    int64_t i = wlo + threadIdx.x;
    for (; i + 3 * 256 < whi; i += 4 * 256) {
        uint4 u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = ((const uint4*)r.base)[i + k * 256];
#pragma unroll
        for (int k = 0; k < 4; ++k) ((uint4*)r.base)[i + k * 256] = scaled(u[k]);
    }
    for (; i < whi; i += 256) ((uint4*)r.base)[i] = scaled(((const uint4*)r.base)[i]);
    auto one = [&](int64_t e) {
        const float v = mt_elem<IS16>(r.base, e) * coef;
        if (IS16) ((__bf16*)r.base)[e] = (__bf16)v;
        else ((float*)r.base)[e] = v;
    };
    if (threadIdx.x < PER && wlo > r.lo) {
        const int64_t e = threadIdx.x;
        if (e >= r.first && e < r.last) one(e);
    }
    if (threadIdx.x < PER && whi < r.hi && whi >= wlo) {
        const int64_t e = whi * PER + threadIdx.x;
        if (e < r.last) one(e);
    }
}
template <bool MAX>
__global__ __launch_bounds__(256) void multi_clip_kernel(const MtList l, const double* __restrict__ partial, int np, float* __restrict__ out,
                                                         const float* __restrict__ norm, float max_norm) {
    const float n = norm != nullptr ? norm[0] : mt_norm<MAX, 256>(partial, np);
    if (out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) out[0] = n;
    float coef = max_norm / (n + 1e-6f);
    coef = coef > 1.f ? 1.f : coef;                // a norm that is no number makes every gradient none, as torch's clipping does
    if (coef == 1.f) return;                       // times one: the gradients are what they would become
    const MtRun r = mt_run(l, gridDim.x - 1 - blockIdx.x);
    if (r.is16) mt_scale<true>(r, coef);
    else mt_scale<false>(r, coef);
}

#include <algorithm>
#include <new>
#include <utility>
#include <vector>
extern "C" int64_t uem_multi_norm_workspace_doubles(int count) { return MT_BLOCKS + 2 * (int64_t)(count > 0 ? count : 0); }
static int multi_lists(const uint64_t* ptrs, const int64_t* numels, const uint8_t* bf16, int count, std::vector<MtList>& lists, int& blocks) {
    int64_t total = 0;
    for (int i = 0; i < count; ++i) {
        UEM_REQUIRE(numels[i] >= 0 && (numels[i] == 0 || ptrs[i] != 0), "multi_norm: tensor %d has %lld elements at %p", i, (long long)numels[i], (void*)ptrs[i]);
        UEM_REQUIRE(ptrs[i] % (bf16[i] ? 2 : 4) == 0, "multi_norm: tensor %d does not begin on an element boundary", i);
        total += numels[i] * (bf16[i] ? 2 : 4);
    }
    // a run of accesses a block: at least four a thread (a small list is over in one round), at most MT_BLOCKS blocks beside those a tensor's ends add
    const int64_t run64 = std::max<int64_t>(1024, uem_cdiv(uem_cdiv(total, 16), MT_BLOCKS));
    UEM_REQUIRE(run64 < ((int64_t)1 << 31), "multi_norm: %lld bytes are more than the kernels cover", (long long)total);
    blocks = 0;
    for (int i = 0; i < count; ++i) {
        if (numels[i] == 0) continue;
        const int size = bf16[i] ? 2 : 4;
        const int64_t accesses = uem_cdiv((int64_t)(ptrs[i] & 15) + numels[i] * size, 16), nb = uem_cdiv(accesses, run64);
        if (lists.empty() || lists.back().count == MT_MOST || lists.back().start[lists.back().count] + nb > 0xffff) {
            lists.emplace_back();
            MtList& l = lists.back();
            l.count = 0; l.part0 = blocks; l.run = (int)run64; l.start[0] = 0;
            for (unsigned& b : l.bf16) b = 0;
        }
        MtList& l = lists.back();
        const int t = l.count++;
        l.ptr[t] = (void*)ptrs[i]; l.n[t] = numels[i];
        if (bf16[i]) l.bf16[t >> 5] |= 1u << (t & 31);
        l.start[t + 1] = (uint16_t)(l.start[t] + nb);
        blocks += (int)nb;
    }
    return UEM_OK;
}
static int multi_run(const uint64_t* ptrs, const int64_t* numels, const uint8_t* bf16, int count, int norm_type, double* partial, float* norm_out,
                     bool clip, float max_norm, hipStream_t st) {
    UEM_REQUIRE(count >= 0 && (count == 0 || (ptrs && numels && bf16)) && partial && norm_out, "multi_norm: bad arguments");
    UEM_REQUIRE(norm_type == 2 || norm_type == 0, "multi_norm: norm type must be 2, or 0 for the largest magnitude");
    std::vector<MtList> lists;
    int blocks = 0;
    const int rc = multi_lists(ptrs, numels, bf16, count, lists, blocks);
    if (rc != UEM_OK) return rc;
    if (clip) {                                    // scaled in place by blocks that know nothing of each other
        std::vector<std::pair<uint64_t, uint64_t>> spans;
        for (int i = 0; i < count; ++i)
            if (numels[i] > 0) spans.emplace_back(ptrs[i], ptrs[i] + (uint64_t)numels[i] * (bf16[i] ? 2 : 4));
        std::sort(spans.begin(), spans.end());
        for (size_t i = 1; i < spans.size(); ++i)
            UEM_REQUIRE(spans[i].first >= spans[i - 1].second, "multi_clip: two of the tensors share memory (0x%llx)", (unsigned long long)spans[i].first);
    }
    const bool mx = norm_type == 0;
    for (const MtList& l : lists) {
        const int nb = l.start[l.count];
        if (mx) multi_norm_partial_kernel<true><<<nb, 256, 0, st>>>(l, partial);
        else multi_norm_partial_kernel<false><<<nb, 256, 0, st>>>(l, partial);
    }
    const bool join = clip && blocks <= MT_JOIN && !lists.empty();
    if (!join) {
        if (mx) multi_norm_final_kernel<true><<<1, 1024, 0, st>>>(partial, blocks, norm_out);
        else multi_norm_final_kernel<false><<<1, 1024, 0, st>>>(partial, blocks, norm_out);
    }
    for (size_t i = clip ? lists.size() : 0; i-- > 0;) {
        const MtList& l = lists[i];
        const int nb = l.start[l.count];
        float* const out = i == 0 && join ? norm_out : nullptr;
        const float* const norm = join ? nullptr : norm_out;
        if (mx) multi_clip_kernel<true><<<nb, 256, 0, st>>>(l, partial, blocks, out, norm, max_norm);
        else multi_clip_kernel<false><<<nb, 256, 0, st>>>(l, partial, blocks, out, norm, max_norm);
    }
    return uem_check_launch("multi_norm");
}
extern "C" int uem_multi_norm(const uint64_t* ptrs, const int64_t* numels, const uint8_t* bf16, int count, int norm_type, double* partial,
                              float* norm_out, void* stream) {
    try {
        return multi_run(ptrs, numels, bf16, count, norm_type, partial, norm_out, false, 0.f, (hipStream_t)stream);
    } catch (const std::bad_alloc&) {
        return uem_fail(UEM_ERR_INVALID, "multi_norm: out of host memory for a list of %d tensors", count);
    }
}
extern "C" int uem_multi_clip(const uint64_t* ptrs, const int64_t* numels, const uint8_t* bf16, int count, int norm_type, double* partial,
                              float* norm_out, float max_norm, void* stream) {
    try {
        return multi_run(ptrs, numels, bf16, count, norm_type, partial, norm_out, true, max_norm, (hipStream_t)stream);
    } catch (const std::bad_alloc&) {
        return uem_fail(UEM_ERR_INVALID, "multi_clip: out of host memory for a list of %d tensors", count);
    }
}
