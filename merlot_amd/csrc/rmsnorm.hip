// Root-mean-square norm for gfx950, forward (with the residual's addition and an 8-bit copy of the output) and backward.
//
//   h = round(x + residual);  R = 1 / sqrt(mean(h^2) + eps);  y = h * R * gamma
//   n = h * R;  t = dy * gamma;  dx = R * (t - n * mean(t * n)) (+ dres);  dgamma += sum over rows of dy * n
//
// Both directions are bound by memory: every operand crosses it once.  A row is held in registers by 4 ... 64 lanes of a wave (up to 2 048 features) or by
// four waves, each lane VEC consecutive features per slab, so a lane's loads and stores are 8 or 16 bytes and the 128 features that share a scale lie in 128 / VEC
// neighbouring lanes.
// Measured (101376 x 768 bf16): forward with residual 117 us = 5.3 TB/s (a large copy: 4.85 TB/s), with the 8-bit copy in place of y 103 us, backward with
// the residual stream's gradient 122 us with dgamma = 5.1 TB/s.  Widths that are whole slabs take code without per-element branches (FULL: backward 184 -> 120 us).
// All sums are fp32.  The statistics are taken from h AS STORED (rounded to its type), so that the backward, which reads the stored h, differentiates the
// function the forward computed.  A finite row has its norm whatever its magnitude: where the squares leave fp32's range the row is scaled first (rms_scaled).
#include "common.h"
#include "blocks8.h"

namespace {

// VEC consecutive elements at any element alignment (gfx950 loads and stores global dwords at byte alignment): rows of odd width need no path of their own
template <typename T, int VEC> struct ElemVec { typedef T type __attribute__((ext_vector_type(VEC), aligned(sizeof(T)))); };

// Elements c ... c + VEC - 1 of a row of H; those past its end are zeros and are not stored.  FULL: H is a whole number of slabs.  base: the slab's first element, the same
// in every lane.  In the slab that the row's end lies in the lane at the end loads the row's last VEC elements and moves them down, and
// a row's loads come before all conversions, so that they are in flight together (element by element, 100000 x 500 bf16 backward: 177 us, this way 89).
template <typename T, int VEC, bool FULL, int SLAB>
__device__ __forceinline__ void load_raw(const T* row, int base, int c, int H, typename ElemVec<T, VEC>::type& t) {
    typedef typename ElemVec<T, VEC>::type vec_t;
    if (FULL) {
        t = *reinterpret_cast<const vec_t*>(row + c);
    } else if (SLAB > 128 && base < H && H >= VEC) {     // lanes behind the end read the row's start: a branch around the load would wait for what is in flight (50000 x 2000
        t = *reinterpret_cast<const vec_t*>(row + (H - c >= VEC ? c : c < H ? H - VEC : 0));     // bf16 backward 250 us, without 165), but pays in narrow rows (x 8: 9.6 us, with 7.7)
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) t[e] = (T)0.f;
        if (H >= VEC) {
            if (c < H) t = *reinterpret_cast<const vec_t*>(row + min(c, H - VEC));
        } else {                                         // a row shorter than a vector
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (c + e < H) t[e] = row[c + e];
        }
    }
}
template <typename T, int VEC, bool FULL, int SLAB>
__device__ __forceinline__ void expand(const typename ElemVec<T, VEC>::type& t, int base, int c, int H, float (&v)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = (float)t[e];
    if (FULL || base + SLAB <= H || H < VEC) return;
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = c < H ? v[e] : 0.f;
    const int s = -H & (VEC - 1);                        // by how much: the same in every row
    const bool end = c < H && H - c < VEC;
#pragma unroll
    for (int b = 1; b < VEC; b *= 2)
        if (s & b)
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = end ? (e + b < VEC ? v[e + b] : 0.f) : v[e];
}
template <typename T, int VEC, bool FULL, int SLAB>
__device__ __forceinline__ void load_vec(const T* row, int base, int c, int H, float (&v)[VEC]) {
    typename ElemVec<T, VEC>::type t;
    load_raw<T, VEC, FULL, SLAB>(row, base, c, H, t);
    expand<T, VEC, FULL, SLAB>(t, base, c, H, v);
}
template <typename T, int VEC, bool FULL, int SLAB>
__device__ __forceinline__ void store_vec(T* row, int base, int c, int H, const float (&v)[VEC]) {
    typedef typename ElemVec<T, VEC>::type vec_t;
    vec_t t;
#pragma unroll
    for (int e = 0; e < VEC; ++e) t[e] = (T)v[e];
    if (FULL || base + SLAB <= H || H - c >= VEC) {
        *reinterpret_cast<vec_t*>(row + c) = t;
    } else if (H > c) {                                  // the end of the row: four, two, one
        const int left = H - c;
        T* p = row + c;
#pragma unroll
        for (int b = VEC / 2; b > 0; b /= 2)
            if (left & b) {
#pragma unroll
                for (int e = 0; e < VEC / 2; ++e)
                    if (e < b) p[e] = t[e];
#pragma unroll
                for (int e = 0; e + b < VEC; ++e) t[e] = t[e + b];
                p += b;
            }
    }
}

// A row's lanes (LPR: lanes per row, 4 ... 256): up to 64 rows share a workgroup.
template <int LPR> struct RowShape {
    static constexpr int WPR = LPR >= 64 ? LPR / 64 : 1, RPW = LPR >= 64 ? 1 : 64 / LPR, RPB = 4 / WPR * RPW;     // waves per row, rows per wave, rows per workgroup
    static __device__ __forceinline__ int lane() { return LPR >= 64 ? (int)threadIdx.x % LPR : (int)threadIdx.x & (LPR - 1); }
    static __device__ __forceinline__ int slot() { return (int)threadIdx.x / LPR; }
};

// sum over the row's WPR waves.  slot: which of the alternating LDS rows this call uses -- a wave may be one call ahead of another, never two.
template <int LPR>
__device__ __forceinline__ float row_sum(float s, float (*red)[RowShape<LPR>::WPR], int& slot) {
    constexpr int WPR = RowShape<LPR>::WPR;
#pragma unroll
    for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if constexpr (WPR > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) red[slot][wave] = s;
        __syncthreads();
        s = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) s += red[slot][w];
        slot ^= 1;
    }
    return s;
}

// largest value of the row's lanes (bit patterns of non-negative floats), the same in each of them; slot: as row_sum
template <int LPR>
__device__ __forceinline__ uint32_t row_umax(uint32_t m, float (*red)[RowShape<LPR>::WPR], int& slot) {
    constexpr int WPR = RowShape<LPR>::WPR;
#pragma unroll
    for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
    if constexpr (WPR > 1) {
        if ((threadIdx.x & 63) == 0) red[slot][threadIdx.x >> 6] = __uint_as_float(m);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WPR; ++w) m = max(m, __float_as_uint(red[slot][w]));
        slot ^= 1;
    }
    return m;
}

// A finite row whose sum of squares leaves fp32 (over 3.4e38, or, with an eps to match, so small that squares lose bits): its values are scaled by a power of two that
// brings the larger of max |v| and sqrt(eps) near 1, and the sum is taken again.  -> 1 / rms of the SCALED row; scale times that is 1 / rms.  Uniform over a row's lanes.
template <int VEC, int NS, int LPR>
__device__ __forceinline__ float rms_scaled(float (&v)[NS][VEC], float& scale, int H, float eps, float (*red)[RowShape<LPR>::WPR], int& slot) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = max(m, __float_as_uint(v[i][e]) & 0x7fffffffu);
    m = row_umax<LPR>(m, red, slot);
    scale = 1.f;
    if (m <= 0x7f7fffffu) {                              // (with an infinity or NaN in the row the sum stays what it is)
        const int e = min(max((int)(max(m, __float_as_uint(sqrtf(fabsf(eps)))) >> 23), 1), 253);
        scale = __uint_as_float((uint32_t)(254 - e) << 23);
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            v[i][e] *= scale;
            ss += v[i][e] * v[i][e];
        }
    ss = row_sum<LPR>(ss, red, slot);
    return 1.0f / sqrtf(ss / (float)H + eps * scale * scale);
}

struct RmsFwdArgs {
    const void* x; int64_t ldx;
    const void* res; int64_t ldr;
    const float* gamma;
    void *h, *y;                 // dense [rows, H]; h only with res
    float* rstd;
    uint8_t* y8; int64_t ld8;    // dense columns up to whole blocks of 128
    uint8_t* s8; int64_t lds8;
    int64_t rows; int H; float eps;
};

template <typename T, int VEC, int NS, int LPR, bool FULL, bool RES>
__global__ __launch_bounds__(256) void rms_fwd_kernel(const RmsFwdArgs p) {
    constexpr int RPB = RowShape<LPR>::RPB, SLAB = LPR * VEC;
    __shared__ float red[2][RowShape<LPR>::WPR];
    int slot = 0;
    const int c0 = RowShape<LPR>::lane() * VEC;          // this lane's first feature of a slab
    const int H = p.H;
    const T* x = (const T*)p.x;
    const T* res = (const T*)p.res;
    for (int64_t row = (int64_t)blockIdx.x * RPB + RowShape<LPR>::slot(); row < p.rows; row += (int64_t)gridDim.x * RPB) {
        float v[NS][VEC];
        float ss = 0.f;
        typename ElemVec<T, VEC>::type tx[NS], tr[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            load_raw<T, VEC, FULL, SLAB>(x + row * p.ldx, i * SLAB, i * SLAB + c0, H, tx[i]);
            if constexpr (RES) load_raw<T, VEC, FULL, SLAB>(res + row * p.ldr, i * SLAB, i * SLAB + c0, H, tr[i]);
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int c = i * SLAB + c0;
            expand<T, VEC, FULL, SLAB>(tx[i], i * SLAB, c, H, v[i]);
            if constexpr (RES) {
                float r[VEC];
                expand<T, VEC, FULL, SLAB>(tr[i], i * SLAB, c, H, r);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[i][e] = (float)(T)(v[i][e] + r[e]);
                store_vec<T, VEC, FULL, SLAB>((T*)p.h + row * H, i * SLAB, c, H, v[i]);
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) ss += v[i][e] * v[i][e];
        }
        ss = row_sum<LPR>(ss, red, slot);
        const float ms = ss / (float)H + p.eps;
        float rstd = 1.0f / sqrtf(ms), scale = 1.f;
        if (!(ms >= 0x1p-90f && ms <= 3.402823466e38f)) rstd = rms_scaled<VEC, NS, LPR>(v, scale, H, p.eps, red, slot);
        if (p.rstd && c0 == 0) p.rstd[row] = rstd * scale;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int c = i * SLAB + c0;
            float g[VEC];
            load_vec<float, VEC, FULL, SLAB>(p.gamma, i * SLAB, c, H, g);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = v[i][e] * rstd * g[e];
            if (p.y) store_vec<T, VEC, FULL, SLAB>((T*)p.y + row * H, i * SLAB, c, H, v[i]);
            if constexpr (SLAB >= 128) {
                if (p.y8) {                                  // from the unrounded y: ONE rounding between it and the 8-bit value
                    uint32_t m = 0;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) m = max(m, __float_as_uint(v[i][e]) & 0x7fffffffu);
                    m = group_umax<128 / VEC>(m);
                    const int byte = block_scale_byte(m, E4M3_TOP);
                    if (FULL || c < p.ld8) {
                        store_codes<0, VEC>(p.y8 + row * p.ld8 + c, v[i], byte);
                        if ((c & 127) == 0) p.s8[row * p.lds8 + (c >> 7)] = (uint8_t)byte;
                    }
                }
            }
        }
    }
}

struct RmsBwdArgs {
    const void* dy; int64_t lddy;
    const void* h; int64_t ldh;
    const float *rstd, *gamma;
    const void* dres; int64_t lddr;
    void* dx;                    // dense [rows, H]
    float* part;                 // [gridDim.x, H]: each workgroup's sums of dy * n
    int64_t rows; int H;
};

template <typename T, int VEC, int NS, int LPR, bool FULL>
__global__ __launch_bounds__(256) void rms_bwd_kernel(const RmsBwdArgs p) {
    // dres is asked for with the other operands where a lane holds much of a row (few waves fit a CU); with less the registers cost more waves than it gains (us, late : early,
    // bf16: 20000 x 5000 222 : 169, 50000 x 2000 182 : 165, 10000 x 8192 150 : 136; 20000 x 4096 126 : 139, 101376 x 768 122 : 128)
    constexpr bool EARLY = NS * VEC >= 24;
    constexpr int RPB = RowShape<LPR>::RPB, SLAB = LPR * VEC;
    __shared__ float red[2][RowShape<LPR>::WPR];
    __shared__ float gred[RPB > 1 ? RPB : 1][RPB > 1 ? SLAB : 1];
    int slot = 0;
    const int c0 = RowShape<LPR>::lane() * VEC;
    const int H = p.H;
    const T* dy = (const T*)p.dy;
    const T* h = (const T*)p.h;
    const T* dres = (const T*)p.dres;
    float dg[NS][VEC];
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) dg[i][e] = 0.f;
    for (int64_t row = (int64_t)blockIdx.x * RPB + RowShape<LPR>::slot(); row < p.rows; row += (int64_t)gridDim.x * RPB) {
        const float rs = p.rstd[row];
        float n[NS][VEC], t[NS][VEC];
        float c1 = 0.f;
        typename ElemVec<T, VEC>::type th[NS], td[NS], te[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            load_raw<T, VEC, FULL, SLAB>(h + row * p.ldh, i * SLAB, i * SLAB + c0, H, th[i]);
            load_raw<T, VEC, FULL, SLAB>(dy + row * p.lddy, i * SLAB, i * SLAB + c0, H, td[i]);
            if (EARLY && dres) load_raw<T, VEC, FULL, SLAB>(dres + row * p.lddr, i * SLAB, i * SLAB + c0, H, te[i]);
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int c = i * SLAB + c0;
            float g[VEC];
            expand<T, VEC, FULL, SLAB>(th[i], i * SLAB, c, H, n[i]);
            expand<T, VEC, FULL, SLAB>(td[i], i * SLAB, c, H, t[i]);
            load_vec<float, VEC, FULL, SLAB>(p.gamma, i * SLAB, c, H, g);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                n[i][e] *= rs;
                dg[i][e] += t[i][e] * n[i][e];
                t[i][e] *= g[e];
                c1 += t[i][e] * n[i][e];
            }
        }
        c1 = row_sum<LPR>(c1, red, slot) / (float)H;
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            const int c = i * SLAB + c0;
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = rs * (t[i][e] - n[i][e] * c1);
            if (dres) {
                float r[VEC];
                if (!EARLY) load_raw<T, VEC, FULL, SLAB>(dres + row * p.lddr, i * SLAB, c, H, te[i]);
                expand<T, VEC, FULL, SLAB>(te[i], i * SLAB, c, H, r);
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] += r[e];
            }
            store_vec<T, VEC, FULL, SLAB>((T*)p.dx + row * H, i * SLAB, c, H, o);
        }
    }
    // the workgroup's rows together, in a fixed order; the partial sums are added up by rms_dgamma_kernel (no atomics: the same call gives the same bits)
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int c = i * SLAB + c0;
        if constexpr (RPB > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VEC; ++e) gred[RowShape<LPR>::slot()][c0 + e] = dg[i][e];
            __syncthreads();
            for (int k = threadIdx.x; k < SLAB; k += 256)
                if (i * SLAB + k < H) {
                    float s = 0.f;
#pragma unroll
                    for (int w = 0; w < RPB; ++w) s += gred[w][k];
                    p.part[(int64_t)blockIdx.x * H + i * SLAB + k] = s;
                }
        } else {
            store_vec<float, VEC, FULL, SLAB>(p.part + (int64_t)blockIdx.x * H, i * SLAB, c, H, dg[i]);
        }
    }
}

// dgamma[c] += sum over the nb partial rows, COLS columns x 1024 / COLS row groups per workgroup: 16 up to 2 048 features, so that enough CUs take part, 64 above (whole backward, 64 : 16
// columns: 8000 x 768 16.1 : 15.2 us, 4099 x 1001 18.8 : 17.4; 8192 x 8192 112 : 116)
template <int COLS>
__global__ __launch_bounds__(1024) void rms_dgamma_kernel(const float* __restrict__ part, float* __restrict__ dgamma, int nb, int H) {
    __shared__ float red[16][COLS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = threadIdx.x % COLS, col = blockIdx.x * COLS + c;
    float s = 0.f;
    if (col < H) {
#pragma unroll 8
        for (int r = threadIdx.x / COLS; r < nb; r += 1024 / COLS) s += part[(int64_t)r * H + col];
    }
#pragma unroll
    for (int o = COLS; o < 64; o *= 2) s += __shfl_xor(s, o, 64);
    if (lane < COLS) red[wave][c] = s;
    __syncthreads();
    if (threadIdx.x < COLS && col < H) {
        s = red[0][c];
#pragma unroll
        for (int w = 1; w < 16; ++w) s += red[w][c];
        dgamma[col] += s;
    }
}

constexpr int RMS_MAX_H = 16384;

// (VEC, slabs, lanes per row) by width.  8 features per lane, 4 where 8 would leave half of the last slab's lanes idle (up to 256 and 768); several rows per wave up to 128
// (200000 x 64 bf16, a wave per row : eight rows: forward 51 : 17 us, backward 84 : 21), four waves per row above 2 048.  narrow: not with the 8-bit copy, whose blocks of 128 are a row's own sixteen lanes
#define RMS_WIDTH(H, V, N, L, ...)                                                                             \
    do {                                                                                                        \
        constexpr int VEC = V, NS = N, LPR = L;                                                                 \
        if ((H) == VEC * LPR * NS) { constexpr bool FULL = true; __VA_ARGS__; }                                        \
        else { constexpr bool FULL = false; __VA_ARGS__; }                                                             \
    } while (0)
#define RMS_DISPATCH(H, narrow, ...)                                                                           \
    do {                                                                                                        \
        if ((H) <= 32 && (narrow)) RMS_WIDTH(H, 8, 1, 4, __VA_ARGS__);                                                 \
        else if ((H) <= 64 && (narrow)) RMS_WIDTH(H, 8, 1, 8, __VA_ARGS__);                                            \
        else if ((H) <= 128) RMS_WIDTH(H, 8, 1, 16, __VA_ARGS__);                                                      \
        else if ((H) <= 256) RMS_WIDTH(H, 4, 1, 64, __VA_ARGS__);                                                      \
        else if ((H) <= 512) RMS_WIDTH(H, 8, 1, 64, __VA_ARGS__);                                                      \
        else if ((H) <= 768) RMS_WIDTH(H, 4, 3, 64, __VA_ARGS__);                                                      \
        else if ((H) <= 1024) RMS_WIDTH(H, 8, 2, 64, __VA_ARGS__);                                                     \
        else if ((H) <= 1536) RMS_WIDTH(H, 8, 3, 64, __VA_ARGS__);                                                     \
        else if ((H) <= 2048) RMS_WIDTH(H, 8, 4, 64, __VA_ARGS__);                                                     \
        else if ((H) <= 4096) RMS_WIDTH(H, 8, 2, 256, __VA_ARGS__);                                                    \
        else if ((H) <= 6144) RMS_WIDTH(H, 8, 3, 256, __VA_ARGS__);                                                    \
        else if ((H) <= 8192) RMS_WIDTH(H, 8, 4, 256, __VA_ARGS__);                                                    \
        else RMS_WIDTH(H, 8, 8, 256, __VA_ARGS__);                                                                     \
    } while (0)

int rms_rows_per_block(int H, bool narrow) { return H <= 32 && narrow ? 64 : H <= 64 && narrow ? 32 : H <= 128 ? 16 : H <= 2048 ? 4 : 1; }

// 1 024 workgroups: 101376 x 768 takes 160 us with 512, 121 with 1 024, 134 with 2 048 (more partial rows to write and add up)
int rms_bwd_blocks(int64_t rows, int H) {
    const int64_t rpb = rms_rows_per_block(H, true), nb = (rows + rpb - 1) / rpb;
    return (int)(nb < 1024 ? nb : 1024);
}

template <typename T>
void rms_fwd_launch(const RmsFwdArgs& a, hipStream_t s) {
    const bool narrow = !a.y8;
    const int64_t rpb = rms_rows_per_block(a.H, narrow), nb = (a.rows + rpb - 1) / rpb;
    const dim3 grid((unsigned)(nb < 4096 ? nb : 4096)), block(256);
    if (a.res)
        RMS_DISPATCH(a.H, narrow, hipLaunchKernelGGL((rms_fwd_kernel<T, VEC, NS, LPR, FULL, true>), grid, block, 0, s, a));
    else
        RMS_DISPATCH(a.H, narrow, hipLaunchKernelGGL((rms_fwd_kernel<T, VEC, NS, LPR, FULL, false>), grid, block, 0, s, a));
}

}  // namespace

extern "C" int merlot_rms_fwd(const void* x, int64_t ldx, int x_f32, const void* residual, int64_t ldr, const float* gamma, void* h, void* y, float* rstd,
                              void* y8, int64_t ld8, uint8_t* scale8, int64_t ld_scale8, int64_t rows, int H, float eps, merlot_stream_t stream) {
    MERLOT_CHECK(x && gamma && (y || y8), MERLOT_ESHAPE, "merlot_rms_fwd: null operand");
    MERLOT_CHECK(rows > 0, MERLOT_ESHAPE, "merlot_rms_fwd: rows must be > 0");
    MERLOT_CHECK(H > 0 && H <= RMS_MAX_H, MERLOT_ESHAPE, "merlot_rms_fwd: H=%d unsupported (1 ... %d)", H, RMS_MAX_H);
    MERLOT_CHECK(ldx >= H && (!residual || ldr >= H), MERLOT_ESHAPE, "merlot_rms_fwd: row stride smaller than H");
    MERLOT_CHECK((residual != nullptr) == (h != nullptr), MERLOT_ESHAPE, "merlot_rms_fwd: h is written with a residual, and only then");
    const int64_t Hp = (H + 127) / 128 * 128;
    MERLOT_CHECK(!y8 || (scale8 && ld8 == Hp && ld_scale8 >= Hp / 128), MERLOT_ESHAPE, "merlot_rms_fwd: the 8-bit copy has ceil(H / 128) * 128 columns and a scale per 128");
    MERLOT_CHECK(!y8 || ((uintptr_t)y8 & 7) == 0, MERLOT_EALIGN, "merlot_rms_fwd: the 8-bit copy must be 8-byte aligned");
    const RmsFwdArgs a = {x, ldx, residual, ldr, gamma, h, y, rstd, (uint8_t*)y8, Hp, scale8, ld_scale8, rows, H, eps};
    if (x_f32) rms_fwd_launch<float>(a, (hipStream_t)stream);
    else rms_fwd_launch<bf16>(a, (hipStream_t)stream);
    return merlot_launch_status("merlot_rms_fwd");
}

extern "C" int64_t merlot_rms_bwd_workspace_bytes(int64_t rows, int H) {
    if (rows <= 0 || H <= 0 || H > RMS_MAX_H) return 0;
    return (int64_t)rms_bwd_blocks(rows, H) * H * 4;
}

extern "C" int merlot_rms_bwd(const void* dy, int64_t lddy, int is_f32, const void* h, int64_t ldh, const float* rstd, const float* gamma, const void* dres,
                              int64_t lddr, void* dx, float* dgamma, int64_t rows, int H, void* workspace, int64_t workspace_bytes, merlot_stream_t stream) {
    MERLOT_CHECK(dy && h && rstd && gamma && dx && dgamma, MERLOT_ESHAPE, "merlot_rms_bwd: null operand");
    MERLOT_CHECK(rows > 0, MERLOT_ESHAPE, "merlot_rms_bwd: rows must be > 0");
    MERLOT_CHECK(H > 0 && H <= RMS_MAX_H, MERLOT_ESHAPE, "merlot_rms_bwd: H=%d unsupported (1 ... %d)", H, RMS_MAX_H);
    MERLOT_CHECK(lddy >= H && ldh >= H && (!dres || lddr >= H), MERLOT_ESHAPE, "merlot_rms_bwd: row stride smaller than H");
    MERLOT_CHECK(workspace && workspace_bytes >= merlot_rms_bwd_workspace_bytes(rows, H), MERLOT_ESHAPE, "merlot_rms_bwd: workspace too small");
    const int nb = rms_bwd_blocks(rows, H);
    const RmsBwdArgs a = {dy, lddy, h, ldh, rstd, gamma, dres, lddr, dx, (float*)workspace, rows, H};
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(nb), block(256);
    if (is_f32) RMS_DISPATCH(H, true, hipLaunchKernelGGL((rms_bwd_kernel<float, VEC, NS, LPR, FULL>), grid, block, 0, s, a));
    else RMS_DISPATCH(H, true, hipLaunchKernelGGL((rms_bwd_kernel<bf16, VEC, NS, LPR, FULL>), grid, block, 0, s, a));
    if (int rc = merlot_launch_status("merlot_rms_bwd")) return rc;
    if (H <= 2048) hipLaunchKernelGGL(rms_dgamma_kernel<16>, dim3((H + 15) / 16), dim3(1024), 0, s, (const float*)workspace, dgamma, nb, H);
    else hipLaunchKernelGGL(rms_dgamma_kernel<64>, dim3((H + 63) / 64), dim3(1024), 0, s, (const float*)workspace, dgamma, nb, H);
    return merlot_launch_status("merlot_rms_bwd");
}
