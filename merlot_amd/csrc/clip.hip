// The global norm of many tensors and the clipped copies of them, for gfx950.
//
//   N = sqrt(sum over tensors and elements of g^2)      out = g * (clip / max(N, clip))
//
// Two passes over the gradients (no element can be scaled before the last one is summed), both bound by memory, in two launches per 128 tensors: the tensors'
// addresses and sizes travel as kernel arguments -- no table in device memory, nothing to copy, nothing kept from one call for the next, and a captured call
// replays as it is.  Squares are summed in 64 bits (a model's 2 * 10^8 addends; half the fp32 rate is far above what memory delivers) in a fixed order: each
// workgroup leaves one partial, every workgroup of the second pass adds all partials up by itself (at most 16 KiB per 128 tensors, from the L2), which saves the
// launch between the passes.  The second pass walks the chunks backwards: what the first pass read last is still in the memory-side cache.
#include <stdlib.h>
#include <algorithm>
#include "common.h"

namespace {

constexpr int CLIP_TENSORS = 128;                        // tensors per launch: 128 x (address, address, size, first chunk) = 3.6 KiB of arguments
constexpr int CLIP_GROUPS = 2048;                        // 16-byte groups of the input per chunk (32 KiB)
constexpr int CLIP_BLOCKS = 2048;                        // workgroups (= partials) per launch at most

struct ClipTable {
    const void* in[CLIP_TENSORS];
    void* out[CLIP_TENSORS];
    int64_t n[CLIP_TENSORS];
    uint32_t chunk0[CLIP_TENSORS + 1];                   // first chunk of each tensor; [count] = all chunks
    uint32_t in16[CLIP_TENSORS / 32], out16[CLIP_TENSORS / 32];   // bit: the tensor is bf16
    int count;
};

__device__ __forceinline__ int clip_find(const ClipTable& t, uint32_t chunk) {   // the tensor a chunk belongs to
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.chunk0[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename T> struct Group16 { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)))); };

// elements i0 ... i0 + E - 1 of g as one aligned 16-byte load, those outside [0, n) as zeros
template <typename T, int E = 16 / sizeof(T)>
__device__ __forceinline__ void clip_load(const T* g, int64_t i0, int64_t n, float (&v)[E]) {
    if (i0 >= 0 && i0 + E <= n) {
        const typename Group16<T>::type t = *reinterpret_cast<const typename Group16<T>::type*>(g + i0);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = (float)t[e];
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = (i0 + e >= 0 && i0 + e < n) ? (float)g[i0 + e] : 0.f;
    }
}

// groups start at multiples of 16 bytes of the INPUT: group k holds elements k * E - shift ...
template <typename T>
__device__ __forceinline__ int clip_shift(const void* g) { return (int)(((uintptr_t)g & 15) / sizeof(T)); }

template <typename T>
__device__ __forceinline__ double clip_square_sum(const T* g, int64_t n, uint32_t chunk) {
    constexpr int E = 16 / sizeof(T), U = 4;
    const int shift = clip_shift<T>(g);
    const int64_t first = (int64_t)chunk * CLIP_GROUPS;
    double s = 0.0;
#pragma unroll
    for (int k = 0; k < CLIP_GROUPS / 256; k += U) {
        float v[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) clip_load<T>(g, (first + (k + u) * 256 + threadIdx.x) * E - shift, n, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < E; ++e) s += (double)v[u][e] * (double)v[u][e];
    }
    return s;
}

// sum over the workgroup's 256 threads, the same bits in every thread
__device__ __forceinline__ double block_sum_f64(double s) {
    __shared__ double red[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

__global__ __launch_bounds__(256) void clip_norm_kernel(const ClipTable t, double* __restrict__ part) {
    double s = 0.0;
    for (uint32_t c = blockIdx.x; c < t.chunk0[t.count]; c += gridDim.x) {
        const int i = clip_find(t, c);
        if (t.in16[i >> 5] >> (i & 31) & 1) s += clip_square_sum<bf16>((const bf16*)t.in[i], t.n[i], c - t.chunk0[i]);
        else s += clip_square_sum<float>((const float*)t.in[i], t.n[i], c - t.chunk0[i]);
    }
    s = block_sum_f64(s);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

template <typename TI, typename TO>
__device__ __forceinline__ void clip_scale(const TI* g, TO* out, int64_t n, uint32_t chunk, float coef) {
    constexpr int E = 16 / sizeof(TI), U = 4;
    const int shift = clip_shift<TI>(g);
    const bool wide = ((uintptr_t)(out - shift) & 15) == 0;      // the output's groups are aligned where the input's are
    const int64_t first = (int64_t)chunk * CLIP_GROUPS;
#pragma unroll
    for (int k = 0; k < CLIP_GROUPS / 256; k += U) {
        float v[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) clip_load<TI>(g, (first + (k + u) * 256 + threadIdx.x) * E - shift, n, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i0 = (first + (k + u) * 256 + threadIdx.x) * E - shift;
            if (wide && i0 >= 0 && i0 + E <= n) {
                typedef TO vec_t __attribute__((ext_vector_type(E), aligned(8)));
                vec_t o;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = (TO)(v[u][e] * coef);
                *reinterpret_cast<vec_t*>(out + i0) = o;
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (i0 + e >= 0 && i0 + e < n) out[i0 + e] = (TO)(v[u][e] * coef);
            }
        }
    }
}

// norm (written by the first workgroup of the first launch) and, with clip > 0, the scaled tensors
__global__ __launch_bounds__(256) void clip_scale_kernel(const ClipTable t, const double* __restrict__ part, int nparts, float clip, float* __restrict__ norm) {
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += 256) s += part[i];
    s = block_sum_f64(s);
    const float total = (float)sqrt(s);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = total;
    if (!(clip > 0.f)) return;
    const float coef = clip / (total < clip ? clip : total);     // a NaN norm stays NaN
    const uint32_t chunks = t.chunk0[t.count];
    for (uint32_t k = blockIdx.x; k < chunks; k += gridDim.x) {
        const uint32_t c = chunks - 1 - k;
        const int i = clip_find(t, c);
        const bool in16 = t.in16[i >> 5] >> (i & 31) & 1, out16 = t.out16[i >> 5] >> (i & 31) & 1;
        if (coef == 1.f && t.in[i] == t.out[i]) continue;        // in place and nothing to clip: every element stays as it is
        const uint32_t lc = c - t.chunk0[i];
        if (in16 && out16) clip_scale<bf16, bf16>((const bf16*)t.in[i], (bf16*)t.out[i], t.n[i], lc, coef);
        else if (in16) clip_scale<bf16, float>((const bf16*)t.in[i], (float*)t.out[i], t.n[i], lc, coef);
        else if (out16) clip_scale<float, bf16>((const float*)t.in[i], (bf16*)t.out[i], t.n[i], lc, coef);
        else clip_scale<float, float>((const float*)t.in[i], (float*)t.out[i], t.n[i], lc, coef);
    }
}

struct Span { uint64_t lo, hi; };

}  // namespace

extern "C" int64_t merlot_clip_workspace_bytes(int64_t n) {
    return n <= 0 ? 0 : (n + CLIP_TENSORS - 1) / CLIP_TENSORS * CLIP_BLOCKS * 8;
}

extern "C" int merlot_clip_by_global_norm(const int64_t* in, const int64_t* out, const int64_t* numel, const uint8_t* types, int64_t n, float clip, float* norm,
                                          void* workspace, int64_t workspace_bytes, merlot_stream_t stream) {
    MERLOT_CHECK(n > 0 && in && numel && types && norm, MERLOT_ESHAPE, "merlot_clip_by_global_norm: no tensors, or a null operand");
    MERLOT_CHECK(clip >= 0.f && clip <= 3.402823466e38f, MERLOT_ESHAPE, "merlot_clip_by_global_norm: clip must be 0 (the norm alone) or positive and finite");
    MERLOT_CHECK(clip == 0.f || out, MERLOT_ESHAPE, "merlot_clip_by_global_norm: null operand");
    MERLOT_CHECK(workspace && workspace_bytes >= merlot_clip_workspace_bytes(n), MERLOT_ESHAPE, "merlot_clip_by_global_norm: workspace too small");
    for (int64_t i = 0; i < n; ++i) {
        MERLOT_CHECK(numel[i] >= 0 && numel[i] < ((int64_t)1 << 40), MERLOT_ESHAPE, "merlot_clip_by_global_norm: tensor %lld has a bad size", (long long)i);
        MERLOT_CHECK(types[i] < 4, MERLOT_EDTYPE, "merlot_clip_by_global_norm: tensor %lld has a bad type", (long long)i);
        MERLOT_CHECK(numel[i] == 0 || (in[i] && (clip == 0.f || out[i])), MERLOT_ESHAPE, "merlot_clip_by_global_norm: null tensor %lld", (long long)i);
        const int si = types[i] & 1 ? 2 : 4, so = types[i] & 2 ? 2 : 4;
        MERLOT_CHECK(in[i] % si == 0 && (clip == 0.f || out[i] % so == 0), MERLOT_EALIGN, "merlot_clip_by_global_norm: tensor %lld is not aligned to its type", (long long)i);
    }
    if (clip > 0.f) {
        // an element written twice, or read after it was written, would be scaled twice or raced for: each output is an output once, and shares bytes with
        // no input but its own (of the same type and address: in place)
        Span* sp = (Span*)malloc(sizeof(Span) * (size_t)n);
        Span* si = (Span*)malloc(sizeof(Span) * (size_t)n);
        if (!sp || !si) {
            free(sp); free(si);
            merlot_set_error("merlot_clip_by_global_norm: out of host memory");
            return MERLOT_ELAUNCH;
        }
        int64_t no = 0, ni = 0;
        for (int64_t i = 0; i < n; ++i)
            if (numel[i]) {
                sp[no++] = {(uint64_t)out[i], (uint64_t)out[i] + (uint64_t)numel[i] * (types[i] & 2 ? 2 : 4)};
                if (!(in[i] == out[i] && (types[i] == 0 || types[i] == 3)))
                    si[ni++] = {(uint64_t)in[i], (uint64_t)in[i] + (uint64_t)numel[i] * (types[i] & 1 ? 2 : 4)};
            }
        const auto by_lo = [](const Span& a, const Span& b) { return a.lo < b.lo; };
        std::sort(sp, sp + no, by_lo);
        std::sort(si, si + ni, by_lo);
        bool clash = false;
        for (int64_t k = 1; k < no; ++k) clash |= sp[k].lo < sp[k - 1].hi;
        uint64_t reach = 0;                              // inputs may overlap each other: the furthest end of those that start before an output's end
        for (int64_t k = 0, j = 0; k < no && !clash; ++k) {
            while (j < ni && si[j].lo < sp[k].hi) { reach = std::max(reach, si[j].hi); clash |= si[j].hi > sp[k].lo; ++j; }
            clash |= reach > sp[k].lo;
        }
        free(sp); free(si);
        MERLOT_CHECK(!clash, MERLOT_ESHAPE, "merlot_clip_by_global_norm: outputs overlap each other or another tensor's input (a tensor given twice?)");
    }
    hipStream_t s = (hipStream_t)stream;
    double* part = (double*)workspace;
    const int64_t launches = (n + CLIP_TENSORS - 1) / CLIP_TENSORS;
    int nparts = 0;
    for (int pass = 0; pass < 2; ++pass) {
        for (int64_t l = 0; l < launches; ++l) {
            ClipTable t;
            t.count = 0;
            uint64_t chunks = 0;
            for (int k = 0; k < CLIP_TENSORS / 32; ++k) t.in16[k] = t.out16[k] = 0;
            for (int64_t i = l * CLIP_TENSORS; i < n && i < (l + 1) * CLIP_TENSORS; ++i) {
                if (numel[i] == 0) continue;
                const int k = t.count++;
                const int es = types[i] & 1 ? 2 : 4;
                const uint64_t groups = ((uint64_t)numel[i] * es + ((uint64_t)in[i] & 15) + 15) / 16;
                t.in[k] = (const void*)in[i];
                t.out[k] = clip > 0.f ? (void*)out[i] : nullptr;
                t.n[k] = numel[i];
                t.chunk0[k] = (uint32_t)chunks;
                t.in16[k >> 5] |= (uint32_t)(types[i] & 1) << (k & 31);
                t.out16[k >> 5] |= (uint32_t)((types[i] >> 1) & 1) << (k & 31);
                chunks += (groups + CLIP_GROUPS - 1) / CLIP_GROUPS;
                MERLOT_CHECK(chunks < ((uint64_t)1 << 31), MERLOT_ESHAPE, "merlot_clip_by_global_norm: 64 TiB in one call");
            }
            t.chunk0[t.count] = (uint32_t)chunks;
            const int blocks = (int)std::min<uint64_t>(std::max<uint64_t>(chunks, 1), CLIP_BLOCKS);
            if (pass == 0) {
                hipLaunchKernelGGL(clip_norm_kernel, dim3(blocks), dim3(256), 0, s, t, part + nparts);
                nparts += blocks;
            } else if (clip > 0.f || l == 0) {
                hipLaunchKernelGGL(clip_scale_kernel, dim3(clip > 0.f ? blocks : 1), dim3(256), 0, s, t, (const double*)part, nparts, clip, l == 0 ? norm : nullptr);
            }
            if (int rc = merlot_launch_status("merlot_clip_by_global_norm")) return rc;
        }
    }
    return MERLOT_OK;
}
