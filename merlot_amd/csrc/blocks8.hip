// 8-bit copies with a scale for each block of 128 (blocks8.h), row-wise and transposed, for gfx950.
//
// One workgroup per 128 x 128 tile of x: the tile is read once into registers (thread = 8 columns x 8 consecutive rows), and both copies are written from there --
// row-wise: 8 codes of a row per thread, blocks along the columns; transposed: 8 codes of a column per thread, blocks along the rows, through an LDS image so that
// memory sees whole 128-byte rows.  Bound by memory: 2 (or 4) bytes read, 1 or 2 written per element.
// Measured (32768 x 4096 bf16): both copies 112 us = 4.8 TB/s, the row-wise one alone 76 us = 5.3 TB/s; a large copy reaches 4.85 TB/s.
// tile128: ONE scale for the whole tile (a weight: both orientations then hold the same codes), written for each of its rows.
#include "blocks8.h"

namespace {

struct QuantArgs {
    const void* x; int64_t ldx;
    uint8_t *q, *s;  int64_t ldq, lds;       // [R, ldq = whole blocks of columns], scales [R, lds]
    uint8_t *qt, *st; int64_t ldqt, ldst;    // [C, ldqt = whole blocks of rows], scales [C, ldst]
    int64_t R, C;
    int tc;                                  // tiles along the columns
};

template <typename T, int FMT, bool TILE, bool WIDE>
__global__ __launch_bounds__(256) void quantize_blocks_kernel(const QuantArgs p) {
    constexpr int TOP = FMT == 0 ? E4M3_TOP : E5M2_TOP;
    __shared__ __attribute__((aligned(16))) uint8_t img[128 * 128];
    __shared__ uint32_t cmax[4][128];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t r0 = (int64_t)(blockIdx.x / p.tc) * 128, c0 = (int64_t)(blockIdx.x % p.tc) * 128;
    const int c8 = tid & 15, r8 = tid >> 4;              // columns c8 * 8 ..., rows r8 * 8 ...
    const T* x = (const T*)p.x + r0 * p.ldx + c0;
    const int rows = (int)min((int64_t)128, p.R - r0), cols = (int)min((int64_t)128, p.C - c0);
    T v[8][8];
    // every lane loads -- from x's start where its own eight elements do not all exist --, so that the eight rows are in flight together; the others are set right after
    const int left = cols - c8 * 8;
    if (p.C >= 8) {
        typedef T vec_t __attribute__((ext_vector_type(8), aligned(WIDE ? 16 : sizeof(T))));
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int row = r8 * 8 + r;
            const vec_t t = *reinterpret_cast<const vec_t*>(row < rows && left >= 8 ? x + row * p.ldx + c8 * 8 : (const T*)p.x);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[r][e] = t[e];
        }
    }
    if (left < 8 || r8 * 8 + 8 > rows) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int row = r8 * 8 + r;
            if (row < rows && left >= 8 && p.C >= 8) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[r][e] = row < rows && e < left ? x[row * p.ldx + c8 * 8 + e] : (T)0.f;
        }
    }
    uint32_t rm[8], cm[8];                               // max |x| as bits: non-negative floats order like their bit patterns, infinities and NaN above all numbers
#pragma unroll
    for (int e = 0; e < 8; ++e) cm[e] = 0u;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        uint32_t m = 0u;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t b = __float_as_uint((float)v[r][e]) & 0x7fffffffu;
            m = max(m, b);
            cm[e] = max(cm[e], b);
        }
        rm[r] = group_umax<16>(m);
    }
    if (TILE || p.qt) {                                  // column maxima over the tile's 128 rows
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            cm[e] = max(cm[e], (uint32_t)__shfl_xor((int)cm[e], 16, 64));
            cm[e] = max(cm[e], (uint32_t)__shfl_xor((int)cm[e], 32, 64));
            if (lane < 16) cmax[wave][c8 * 8 + e] = cm[e];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) cm[e] = max(max(cmax[0][c8 * 8 + e], cmax[1][c8 * 8 + e]), max(cmax[2][c8 * 8 + e], cmax[3][c8 * 8 + e]));
        if constexpr (TILE) {
            uint32_t m = 0u;
#pragma unroll
            for (int e = 0; e < 8; ++e) m = max(m, cm[e]);
            m = group_umax<16>(m);                       // a group of 16 lanes holds all 128 columns
#pragma unroll
            for (int e = 0; e < 8; ++e) rm[e] = cm[e] = m;
        }
    }
    if (p.q) {
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const int row = r8 * 8 + r;
            if (row >= rows) continue;
            const int byte = block_scale_byte(rm[r], TOP);
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = (float)v[r][e];
            store_codes<FMT, 8>(p.q + (r0 + row) * p.ldq + c0 + c8 * 8, f, byte);
            if (c8 == 0) p.s[(r0 + row) * p.lds + (c0 >> 7)] = (uint8_t)byte;
        }
    }
    if (p.qt) {
        // image: column c's 128 codes at c * 128, its 16-byte pieces exchanged by c8 so that the lanes' 8-byte writes spread over the banks
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int col = c8 * 8 + e;
            float f[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) f[r] = (float)v[r][e];
            store_codes<FMT, 8>(img + col * 128 + ((((r8 >> 1) ^ c8) & 7) << 4) + (r8 & 1) * 8, f, block_scale_byte(cm[e], TOP));
            if (r8 == 0 && col < cols) p.st[(c0 + col) * p.ldst + (r0 >> 7)] = (uint8_t)block_scale_byte(cm[e], TOP);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int col = k * 32 + (tid >> 3), piece = tid & 7;
            if (col < cols)
                *reinterpret_cast<u32x4*>(p.qt + (c0 + col) * p.ldqt + r0 + piece * 16) =
                    *reinterpret_cast<const u32x4*>(img + col * 128 + (((piece ^ (col >> 3)) & 7) << 4));
        }
    }
}

template <typename T, int FMT>
void quantize_launch(const QuantArgs& a, bool tile, bool wide, dim3 grid, hipStream_t s) {
    const dim3 block(256);
    if (tile) {
        if (wide) hipLaunchKernelGGL((quantize_blocks_kernel<T, FMT, true, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((quantize_blocks_kernel<T, FMT, true, false>), grid, block, 0, s, a);
    } else {
        if (wide) hipLaunchKernelGGL((quantize_blocks_kernel<T, FMT, false, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((quantize_blocks_kernel<T, FMT, false, false>), grid, block, 0, s, a);
    }
}

}  // namespace

extern "C" int merlot_quantize_blocks(const void* x, int64_t ldx, int x_f32, int64_t R, int64_t C, int fmt, int tile, void* q, int64_t ldq, uint8_t* s,
                                      int64_t lds, void* qt, int64_t ldqt, uint8_t* st, int64_t ldst, merlot_stream_t stream) {
    MERLOT_CHECK(x && (q || qt) && (!q || s) && (!qt || st), MERLOT_ESHAPE, "merlot_quantize_blocks: null operand");
    MERLOT_CHECK(R > 0 && C > 0 && ldx >= C, MERLOT_ESHAPE, "merlot_quantize_blocks: empty, or row stride smaller than the row");
    MERLOT_CHECK(fmt == 0 || fmt == 1, MERLOT_EDTYPE, "merlot_quantize_blocks: fmt must be 0 (e4m3) or 1 (e5m2)");
    MERLOT_CHECK(tile == 1 || tile == 128, MERLOT_ESHAPE, "merlot_quantize_blocks: tile must be 1 or 128");
    const int64_t tr = (R + 127) / 128, tc = (C + 127) / 128;
    MERLOT_CHECK(tr * tc < ((int64_t)1 << 24), MERLOT_ESHAPE, "merlot_quantize_blocks: too many tiles");
    MERLOT_CHECK(!q || (ldq >= tc * 128 && ldq % 16 == 0 && lds >= tc), MERLOT_ESHAPE, "merlot_quantize_blocks: the row-wise copy has ceil(C / 128) * 128 columns and a scale per 128");
    MERLOT_CHECK(!qt || (ldqt >= tr * 128 && ldqt % 16 == 0 && ldst >= tr), MERLOT_ESHAPE, "merlot_quantize_blocks: the transposed copy has ceil(R / 128) * 128 columns and a scale per 128");
    MERLOT_CHECK((((uintptr_t)q | (uintptr_t)qt) & 15) == 0, MERLOT_EALIGN, "merlot_quantize_blocks: the copies must be 16-byte aligned");
    const QuantArgs a = {x, ldx, (uint8_t*)q, s, ldq, lds, (uint8_t*)qt, st, ldqt, ldst, R, C, (int)tc};
    const dim3 grid((unsigned)(tr * tc));
    const bool wide = ((uintptr_t)x & 15) == 0 && ldx * (x_f32 ? 4 : 2) % 16 == 0;
    hipStream_t hs = (hipStream_t)stream;
    if (x_f32) {
        if (fmt == 0) quantize_launch<float, 0>(a, tile == 128, wide, grid, hs);
        else quantize_launch<float, 1>(a, tile == 128, wide, grid, hs);
    } else {
        if (fmt == 0) quantize_launch<bf16, 0>(a, tile == 128, wide, grid, hs);
        else quantize_launch<bf16, 1>(a, tile == 128, wide, grid, hs);
    }
    return merlot_launch_status("merlot_quantize_blocks");
}
