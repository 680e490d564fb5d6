// The global norm of many tensors and the clipped copies of them, for gfx950.
//
//   N = sqrt(sum over tensors and elements of g^2)      out = g * (clip / max(N, clip))
//
// Two passes over the gradients (no element can be scaled before the last one is summed), both bound by memory, in two launches: the tensors' addresses and sizes travel
// as kernel arguments, those of more than 112 tensors by way of small launches that write them into a table in the workspace -- nothing to copy, nothing kept from one call
// for the next, and a captured call replays as it is.  Squares are summed in 64 bits (a model's 2 * 10^8 addends; half the fp32 rate is far above what memory
// delivers) in a fixed order: each workgroup leaves one partial, every workgroup of the second pass adds all partials up by itself (8 KiB from the L2), which
// saves the launch between the passes.  Measured: one buffer of 223 M fp32 values 149 us (6.0 TB/s) + 323 us (5.5 TB/s), 300 tensors of 60 M values in all 136 us.
#include <stdlib.h>
#include <algorithm>
#include "common.h"

namespace {

constexpr int CLIP_TENSORS = 112;                        // tensors whose entries fit a launch's arguments: 3.5 KiB
constexpr int CLIP_CHUNK = 4096;                         // elements per chunk, whatever their type: stretches of chunks are equal work
constexpr int CLIP_BLOCKS = 1536;                        // workgroups (= partials) at most

struct ClipEntry {
    const void* in;
    void* out;
    int64_t n;
    uint32_t chunk0;                                     // the tensor's first chunk
    uint32_t types;                                      // bit 0: in is bf16, bit 1: out is bf16
};
struct ClipTable { ClipEntry e[CLIP_TENSORS]; };

__device__ __forceinline__ int clip_find(const ClipEntry* t, int count, uint32_t chunk) {   // the tensor a chunk belongs to
    int lo = 0, hi = count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t[mid].chunk0 <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename T> struct Group16 { typedef T type __attribute__((ext_vector_type(16 / sizeof(T)))); };

// elements i0 ... i0 + E - 1 of g as one aligned 16-byte load, those outside [0, n) as zeros
template <typename T, bool LAST, int E = 16 / sizeof(T)>
__device__ __forceinline__ void clip_load(const T* g, int64_t i0, int64_t n, float (&v)[E]) {
    if (i0 >= 0 && i0 + E <= n) {
        typename Group16<T>::type t;                     // LAST: nobody reads it again -- past the caches (one buffer of 223 M values 479 -> 471 us)
        if constexpr (LAST) t = __builtin_nontemporal_load(reinterpret_cast<const typename Group16<T>::type*>(g + i0));
        else t = *reinterpret_cast<const typename Group16<T>::type*>(g + i0);
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
    constexpr int E = 16 / sizeof(T), U = CLIP_CHUNK / E / 256;
    const int shift = clip_shift<T>(g);
    const int64_t first = (int64_t)chunk * (CLIP_CHUNK / E);
    double s = 0.0;
    float v[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) clip_load<T, false>(g, (first + u * 256 + threadIdx.x) * E - shift, n, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) s += (double)v[u][e] * (double)v[u][e];
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

// a workgroup's chunks: a contiguous stretch, so that it looks its tensor up once and walks on from there
__device__ __forceinline__ void clip_norm(const ClipEntry* t, int count, uint32_t chunks, double* part) {
    uint32_t c = (uint32_t)((uint64_t)chunks * blockIdx.x / gridDim.x);
    const uint32_t end = (uint32_t)((uint64_t)chunks * (blockIdx.x + 1) / gridDim.x);
    double s = 0.0;
    int i = c < end ? clip_find(t, count, c) : 0;
    for (; c < end; ++c) {
        while (i + 1 < count && t[i + 1].chunk0 <= c) ++i;
        const ClipEntry e = t[i];
        if (e.types & 1) s += clip_square_sum<bf16>((const bf16*)e.in, e.n, c - e.chunk0);
        else s += clip_square_sum<float>((const float*)e.in, e.n, c - e.chunk0);
    }
    s = block_sum_f64(s);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}
__global__ __launch_bounds__(256) void clip_norm_kernel(const ClipTable t, int count, uint32_t chunks, double* __restrict__ part) { clip_norm(t.e, count, chunks, part); }
__global__ __launch_bounds__(256) void clip_norm_table_kernel(const ClipEntry* __restrict__ t, int count, uint32_t chunks, double* __restrict__ part) {
    clip_norm(t, count, chunks, part);
}
// up to CLIP_TENSORS entries from the arguments into a table in the workspace
__global__ __launch_bounds__(128) void clip_table_kernel(const ClipTable t, ClipEntry* __restrict__ out, int count) {
    if ((int)threadIdx.x < count) out[threadIdx.x] = t.e[threadIdx.x];
}

template <typename TI, typename TO>
__device__ __forceinline__ void clip_scale(const TI* g, TO* out, int64_t n, uint32_t chunk, float coef) {
    constexpr int E = 16 / sizeof(TI), U = CLIP_CHUNK / E / 256;
    const int shift = clip_shift<TI>(g);
    const int64_t first = (int64_t)chunk * (CLIP_CHUNK / E);
    float v[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) clip_load<TI, true>(g, (first + u * 256 + threadIdx.x) * E - shift, n, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i0 = (first + u * 256 + threadIdx.x) * E - shift;
        if (i0 >= 0 && i0 + E <= n) {
            // whole groups wherever the output starts (gfx950 stores global dwords at byte alignment): 300 outputs packed into one buffer, 60 M values, 188 -> 141 us
            typedef TO vec_t __attribute__((ext_vector_type(E), aligned(sizeof(TO))));
            vec_t o;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = (TO)(v[u][e] * coef);
            // past the caches too, so that the inputs the first pass read last stay there (533 -> 495 us); a lane's two pieces of a wider type are no whole lines
            if constexpr (sizeof(TO) <= sizeof(TI)) __builtin_nontemporal_store(o, reinterpret_cast<vec_t*>(out + i0));
            else *reinterpret_cast<vec_t*>(out + i0) = o;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (i0 + e >= 0 && i0 + e < n) out[i0 + e] = (TO)(v[u][e] * coef);
        }
    }
}

// norm (written by the first workgroup) and, with clip > 0, the scaled tensors
__device__ __forceinline__ void clip_scale_all(const ClipEntry* t, int count, uint32_t chunks, const double* part, int nparts, float clip, float* norm) {
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += 256) s += part[i];
    s = block_sum_f64(s);
    const float total = (float)sqrt(s);
    if (blockIdx.x == 0 && threadIdx.x == 0) norm[0] = total;
    if (!(clip > 0.f)) return;
    const float coef = clip / (total < clip ? clip : total);     // a NaN norm stays NaN
    // the last stretch first: what the first pass read last is still in the memory-side cache
    const uint32_t b = gridDim.x - 1 - blockIdx.x, first = (uint32_t)((uint64_t)chunks * b / gridDim.x);
    uint32_t c = (uint32_t)((uint64_t)chunks * (b + 1) / gridDim.x);
    int i = c > first ? clip_find(t, count, c - 1) : 0;
    while (c > first) {
        --c;
        while (t[i].chunk0 > c) --i;
        const ClipEntry e = t[i];
        if (coef == 1.f && e.in == e.out) continue;              // in place and nothing to clip: every element stays as it is
        const uint32_t lc = c - e.chunk0;
        if (e.types == 3) clip_scale<bf16, bf16>((const bf16*)e.in, (bf16*)e.out, e.n, lc, coef);
        else if (e.types == 1) clip_scale<bf16, float>((const bf16*)e.in, (float*)e.out, e.n, lc, coef);
        else if (e.types == 2) clip_scale<float, bf16>((const float*)e.in, (bf16*)e.out, e.n, lc, coef);
        else clip_scale<float, float>((const float*)e.in, (float*)e.out, e.n, lc, coef);
    }
}
__global__ __launch_bounds__(256) void clip_scale_kernel(const ClipTable t, int count, uint32_t chunks, const double* __restrict__ part, int nparts, float clip,
                                                         float* __restrict__ norm) {
    clip_scale_all(t.e, count, chunks, part, nparts, clip, norm);
}
__global__ __launch_bounds__(256) void clip_scale_table_kernel(const ClipEntry* __restrict__ t, int count, uint32_t chunks, const double* __restrict__ part, int nparts,
                                                               float clip, float* __restrict__ norm) {
    clip_scale_all(t, count, chunks, part, nparts, clip, norm);
}

// chunks of a tensor at that address (groups start at multiples of 16 bytes)
uint64_t clip_chunks(int64_t address, int64_t numel, int size) { return ((uint64_t)numel + ((uint64_t)address & 15) / size + CLIP_CHUNK - 1) / CLIP_CHUNK; }

struct Span { uint64_t lo, hi; };

}  // namespace

extern "C" int64_t merlot_clip_workspace_bytes(int64_t n) {
    return n <= 0 ? 0 : CLIP_BLOCKS * 8 + (n > CLIP_TENSORS ? n * (int64_t)sizeof(ClipEntry) : 0);
}

extern "C" int merlot_clip_by_global_norm(const int64_t* in, const int64_t* out, const int64_t* numel, const uint8_t* types, int64_t n, float clip, float* norm,
                                          void* workspace, int64_t workspace_bytes, merlot_stream_t stream) {
    MERLOT_CHECK(n > 0 && in && numel && types && norm, MERLOT_ESHAPE, "merlot_clip_by_global_norm: no tensors, or a null operand");
    MERLOT_CHECK(clip >= 0.f && clip <= 3.402823466e38f, MERLOT_ESHAPE, "merlot_clip_by_global_norm: clip must be 0 (the norm alone) or positive and finite");
    MERLOT_CHECK(clip == 0.f || out, MERLOT_ESHAPE, "merlot_clip_by_global_norm: null operand");
    MERLOT_CHECK(workspace && workspace_bytes >= merlot_clip_workspace_bytes(n), MERLOT_ESHAPE, "merlot_clip_by_global_norm: workspace too small");
    MERLOT_CHECK(((uintptr_t)workspace & 7) == 0, MERLOT_EALIGN, "merlot_clip_by_global_norm: workspace must be 8-byte aligned");
    uint64_t all = 0;
    for (int64_t i = 0; i < n; ++i) {
        MERLOT_CHECK(numel[i] >= 0 && numel[i] < ((int64_t)1 << 40), MERLOT_ESHAPE, "merlot_clip_by_global_norm: tensor %lld has a bad size", (long long)i);
        MERLOT_CHECK(types[i] < 4, MERLOT_EDTYPE, "merlot_clip_by_global_norm: tensor %lld has a bad type", (long long)i);
        MERLOT_CHECK(numel[i] == 0 || (in[i] && (clip == 0.f || out[i])), MERLOT_ESHAPE, "merlot_clip_by_global_norm: null tensor %lld", (long long)i);
        const int si = types[i] & 1 ? 2 : 4, so = types[i] & 2 ? 2 : 4;
        MERLOT_CHECK(in[i] % si == 0 && (clip == 0.f || out[i] % so == 0), MERLOT_EALIGN, "merlot_clip_by_global_norm: tensor %lld is not aligned to its type", (long long)i);
        if (numel[i]) all += clip_chunks(in[i], numel[i], si);
        MERLOT_CHECK(all < ((uint64_t)1 << 31) && i < (1 << 30), MERLOT_ESHAPE, "merlot_clip_by_global_norm: 2^43 elements or more (each tensor counted in whole 4096s), or 2^30 tensors, in one call");
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
    ClipEntry* table = n > CLIP_TENSORS ? (ClipEntry*)(part + CLIP_BLOCKS) : nullptr;
    ClipTable t;
    int count = 0, filled = 0;                           // entries in all, of them in the workspace's table
    uint64_t chunks = 0;
    for (int64_t i = 0; i < n; ++i) {
        if (numel[i] == 0) continue;
        t.e[count - filled] = {(const void*)in[i], clip > 0.f ? (void*)out[i] : nullptr, numel[i], (uint32_t)chunks, types[i]};
        ++count;
        chunks += clip_chunks(in[i], numel[i], types[i] & 1 ? 2 : 4);
        if (table && count - filled == CLIP_TENSORS) {
            hipLaunchKernelGGL(clip_table_kernel, dim3(1), dim3(128), 0, s, t, table + filled, CLIP_TENSORS);
            filled = count;
        }
    }
    if (table && count > filled) hipLaunchKernelGGL(clip_table_kernel, dim3(1), dim3(128), 0, s, t, table + filled, count - filled);
    const int blocks = (int)std::min<uint64_t>(std::max<uint64_t>(chunks, 1), CLIP_BLOCKS);
    const dim3 grid(blocks), last(clip > 0.f ? blocks : 1), block(256);
    if (table) {
        hipLaunchKernelGGL(clip_norm_table_kernel, grid, block, 0, s, (const ClipEntry*)table, count, (uint32_t)chunks, part);
        hipLaunchKernelGGL(clip_scale_table_kernel, last, block, 0, s, (const ClipEntry*)table, count, (uint32_t)chunks, (const double*)part, blocks, clip, norm);
    } else {
        hipLaunchKernelGGL(clip_norm_kernel, grid, block, 0, s, t, count, (uint32_t)chunks, part);
        hipLaunchKernelGGL(clip_scale_kernel, last, block, 0, s, t, count, (uint32_t)chunks, (const double*)part, blocks, clip, norm);
    }
    return merlot_launch_status("merlot_clip_by_global_norm");
}
