// Matrix product of two 8-bit float operands with a power-of-two scale for each row and block of 128 along the reduction (blocks8.h), for gfx950.
//
//   C[m, n] (+)= sum over blocks b of 2^(ea[m, b] + eb[n, b]) * sum over k in b of A[m, k] * B[n, k]   (+ bias[n])
//
// Two ways to multiply, both with fp32 accumulators:
//   * bf16 outputs: v_mfma_scale_f32_32x32x64_f8f6f4 takes a scale byte per lane -- the row and half K-step the lane holds -- beside the 8-bit operands, so the
//     scales cost nothing.  The instruction adds groups of eight products aligned to the largest of them and keeps 13 bits below it (measured: a product 2^13
//     smaller than another one of its group is lost); on real operands that is 1.3e-5 of the result, 1 / 300 of the output's own rounding.
//   * fp32 outputs (a weight gradient added to others, logits): that would be the largest error there is.  A code times a power of two is a bf16 value, so the
//     fragments are converted exactly (v_cvt_scalef32_pk_bf16_*, the scale included) and go through v_mfma_f32_32x32x16_bf16, whose sums are good to fp32.  Half the
//     matrix rate, still 8-bit traffic.
#include "blocks8.h"

namespace {

struct BlocksArgs {
    const uint8_t *A, *B, *sa, *sb;
    int64_t lda, ldb, ldsa, ldsb;
    void* C; int64_t ldc;
    const float* bias;
    float* part;                             // split reductions: [splits][M][N] partial products
    int64_t M, N;
    int nk, nk_split;                        // blocks of 128 in all, per split
    int ntm, ntn;
    int accumulate;
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const uint8_t* p, int64_t row0, int64_t rows, int64_t ld, int64_t width) {
    // the rows of one tile as a buffer of their own: offsets stay small however large the operand is, and rows past its end read as zeros
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p + row0 * ld), 0, rows > 0 ? (int)((rows - 1) * ld + width) : 0, 0x00020000);
}

// up to E consecutive columns n ... of row m; add: onto what is there (fp32 only)
template <typename T, int E>
__device__ __forceinline__ void store_out(T* C, int64_t ldc, int64_t m, int64_t n, int64_t left, T __attribute__((ext_vector_type(E))) v, bool add) {
    typedef T vec_t __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    T* c = C + m * ldc + n;
    if (left >= E) {
        if constexpr (sizeof(T) == 4)
            if (add) v += *reinterpret_cast<const vec_t*>(c);
        *reinterpret_cast<vec_t*>(c) = v;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (e < left) c[e] = sizeof(T) == 4 && add ? (T)((float)c[e] + (float)v[e]) : v[e];
    }
}

// 2^(byte - 127); 255 is NaN
__device__ __forceinline__ float scale_value(int byte) {
    return __uint_as_float(byte == 255 ? 0x7fc00000u : byte == 0 ? 0x00400000u : (uint32_t)byte << 23);
}

// eight codes -> eight bf16 values, times 2^(byte - 127)
template <int FMT>
__device__ __forceinline__ bf16x8 widen(int lo, int hi, float scale) {
    bf16x8 r;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const unsigned w = (unsigned)(k < 2 ? lo : hi);
        bf16x2 t;
        if constexpr (FMT == 0) t = (k & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false);
        else t = (k & 1) ? __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, false);
        r[2 * k] = t[0];
        r[2 * k + 1] = t[1];
    }
    return r;
}

template <int N>
__device__ __forceinline__ void wait_step() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// Tile 128 x BN, four waves (64 x 128 each for BN 256, 64 x 64 for BN 128), K-steps of 64, three step buffers filled by LDS-DMA two steps ahead, one barrier per
// step.  Two workgroups share a CU (72 + 6 KiB of LDS, 256 registers): while one waits, loads or stores its tile, the other multiplies.
// OUT: 0 bf16, 1 fp32, 2 fp32 partial products of a split reduction.  EXACT: through bf16 fragments (see above).
constexpr int SCALE_BLOCKS = 16;                         // blocks of 128 whose scale bytes lie in LDS at a time (16 bytes per row)

template <int FA, int BN, int OUT, bool EXACT>
__global__ __launch_bounds__(256, 2) void blocks_gemm_kernel(const BlocksArgs p) {
#ifdef __HIP_DEVICE_COMPILE__                            // (with this body in the host pass, the compiler leaves the kernel's launch stub out without a word)
    constexpr int BM = 128, NJ = BN / 64;                // 32-column fragments per wave
    constexpr int STEP = (BM + BN) * 64;                 // bytes of one K-step
    constexpr int PIECES = STEP / 1024 / 4;              // 1-KiB pieces per wave and step
    __shared__ __attribute__((aligned(1024))) uint8_t lds[3 * STEP + (BM + BN) * SCALE_BLOCKS];
    uint8_t* const scales = lds + 3 * STEP;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, l31 = lane & 31, wm = wave >> 1, wn = wave & 1;
    // tiles in bands of eight tile rows, column by column, a contiguous stretch per XCD: the tiles in flight on one XCD share their rows and columns in its L2
    int tm, tn;
    {
        const int nwg = p.ntm * p.ntn, q = nwg >> 3, r = nwg & 7, xcd = (int)blockIdx.x & 7;
        const int id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + ((int)blockIdx.x >> 3);
        const int band = id / (8 * p.ntn), in = id - band * 8 * p.ntn, high = min(8, p.ntm - band * 8);
        tm = band * 8 + in % high;
        tn = in / high;
    }
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN;
    const int kb0 = OUT == 2 ? (int)blockIdx.y * p.nk_split : 0, kb1 = OUT == 2 ? min(p.nk, kb0 + p.nk_split) : p.nk;
    const int rows_a = (int)min((int64_t)BM, p.M - m0), rows_b = (int)min((int64_t)BN, p.N - n0);
    const int64_t K = (int64_t)p.nk * 128, sw = (p.nk + 3) & ~3;
    const __amdgpu_buffer_rsrc_t ra = rows_rsrc(p.A, m0, rows_a, p.lda, K), rb = rows_rsrc(p.B, n0, rows_b, p.ldb, K);
    const __amdgpu_buffer_rsrc_t rsa = rows_rsrc(p.sa, m0, rows_a, p.ldsa, sw), rsb = rows_rsrc(p.sb, n0, rows_b, p.ldsb, sw);
    // LDS image of a step: row r (A's, then B's) at r * 64, its 16-byte chunk c at position c ^ ((r >> 2) & 3): sixteen lanes that read sixteen rows at one chunk
    // meet all 64 banks
    unsigned off[PIECES];                                // a wave fetches two pieces of A and the rest of B
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int row = (i < 2 ? wave * 2 + i : wave * (PIECES - 2) + i - 2) * 16 + (lane >> 2), ch = ((lane & 3) ^ (row >> 2)) & 3;
        off[i] = (unsigned)(row * (i < 2 ? p.lda : p.ldb)) + ch * 16;
    }
    auto issue = [&](int step, int buf) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if (i < 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, LDS_PTR(lds + buf * STEP + (wave * 2 + i) * 1024), 16, off[i], step * 64, 0, 0);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, LDS_PTR(lds + buf * STEP + (8 + wave * (PIECES - 2) + i - 2) * 1024), 16, off[i], step * 64, 0, 0);
        }
    };
    // the scale bytes of sixteen blocks from block b on, a word of four blocks per thread and turn (a split starts at a multiple of four blocks)
    auto load_scales = [&](int b) {
#pragma unroll
        for (int k = 0; k < (BM + BN) / 64; ++k) {
            const int row = k * 64 + (tid >> 2), b4 = b + (tid & 3) * 4;
            const int v = k < BM / 64 ? __builtin_amdgcn_raw_buffer_load_b32(rsa, (unsigned)(row * p.ldsa + b4), 0, 0)
                                      : __builtin_amdgcn_raw_buffer_load_b32(rsb, (unsigned)((row - BM) * p.ldsb + b4), 0, 0);
            *reinterpret_cast<int*>(scales + row * 16 + (tid & 3) * 4) = v;
        }
    };
    load_scales(kb0);
    f32x16 acc[2][NJ];                                   // lane <-> row of A, register r <-> column (r & 3) + 8 (r >> 2) + 4 hi of a fragment; they start at the bias
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int64_t n = n0 + wn * (BN / 2) + j * 32 + (r & 3) + 8 * (r >> 2) + 4 * hi;
            acc[0][j][r] = acc[1][j][r] = (OUT != 2 && p.bias && n < p.N) ? p.bias[n] : 0.f;
        }
    unsigned ra_off[2], rb_off[NJ];                      // fragment rows in a step's image, and this lane's pair of chunks (2 hi, 2 hi + 1) there
    unsigned ca[2], cb[NJ];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = wm * 64 + i * 32 + l31;
        ra_off[i] = row * 64;
        ca[i] = ((2 * hi) ^ (row >> 2)) & 3;
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        const int row = BM + wn * (BN / 2) + j * 32 + l31;
        rb_off[j] = row * 64;
        cb[j] = ((2 * hi) ^ (row >> 2)) & 3;
    }
    auto fragment = [&](int buf, unsigned row_off, unsigned c) -> i32x8 {
        const i32x4 x = *reinterpret_cast<const i32x4*>(lds + buf * STEP + row_off + c * 16);
        const i32x4 y = *reinterpret_cast<const i32x4*>(lds + buf * STEP + row_off + (c ^ 1) * 16);
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    const int steps = 2 * (kb1 - kb0);
    issue(2 * kb0, 0);
    issue(2 * kb0 + 1, 1);
    int buf = 0;
    int xa[2], xb[NJ];
    for (int t = 0; t < steps; ++t) {
        // the last words of the old sixteen blocks were read eight steps ago, seven barriers back
        if (t && (t & (2 * SCALE_BLOCKS - 1)) == 0) load_scales(kb0 + (t >> 1));
        if (t + 1 < steps) wait_step<PIECES>();
        else wait_step<0>();
        __builtin_amdgcn_s_barrier();
        if (t + 2 < steps) issue(2 * kb0 + t + 2, buf == 0 ? 2 : buf - 1);
        if ((t & 7) == 0) {                              // four blocks' bytes per word
#pragma unroll
            for (int i = 0; i < 2; ++i) xa[i] = *reinterpret_cast<const int*>(scales + (wm * 64 + i * 32 + l31) * 16 + ((t >> 3) & 3) * 4);
#pragma unroll
            for (int j = 0; j < NJ; ++j) xb[j] = *reinterpret_cast<const int*>(scales + (BM + wn * (BN / 2) + j * 32 + l31) * 16 + ((t >> 3) & 3) * 4);
        } else if ((t & 1) == 0) {
#pragma unroll
            for (int i = 0; i < 2; ++i) xa[i] = (int)((unsigned)xa[i] >> 8);
#pragma unroll
            for (int j = 0; j < NJ; ++j) xb[j] = (int)((unsigned)xb[j] >> 8);
        }
        i32x8 fa[2], fb[NJ];
#pragma unroll
        for (int i = 0; i < 2; ++i) fa[i] = fragment(buf, ra_off[i], ca[i]);
#pragma unroll
        for (int j = 0; j < NJ; ++j) fb[j] = fragment(buf, rb_off[j], cb[j]);
        if constexpr (!EXACT) {
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[j], fa[i], acc[i][j], 0, FA, 0, xb[j], 0, xa[i]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {                // lane k-bytes 8 q ... : the same eight of both operands, which is all a dot product asks for
                bf16x8 wa[2], wb[NJ];
#pragma unroll
                for (int i = 0; i < 2; ++i) wa[i] = widen<FA>(fa[i][2 * q], fa[i][2 * q + 1], scale_value(xa[i] & 255));
#pragma unroll
                for (int j = 0; j < NJ; ++j) wb[j] = widen<0>(fb[j][2 * q], fb[j][2 * q + 1], scale_value(xb[j] & 255));
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j], wa[i], acc[i][j], 0, 0, 0);
            }
        }
        buf = buf == 2 ? 0 : buf + 1;
    }
    // ---- epilogue: 32 rows at a time through a slab of the wave's own in the step buffers, so that memory sees whole rows of the wave's columns
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    typedef typename std::conditional<OUT == 0, bf16, float>::type T;
    constexpr int COLS = BN / 2, LDR = COLS * (int)sizeof(T) + 16, E = 16 / (int)sizeof(T), LPR = COLS / E;      // slab row in bytes; 16-byte groups per row
    static_assert(4 * 32 * LDR <= 3 * STEP, "slabs");
    uint8_t* const slab = lds + wave * 32 * LDR;
    T* const C = OUT == 2 ? (T*)p.part + (int64_t)blockIdx.y * p.M * p.N : (T*)p.C;
    const int64_t ldc = OUT == 2 ? p.N : p.ldc, n = n0 + wn * COLS + (lane % LPR) * E;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                typedef T vec_t __attribute__((ext_vector_type(4)));
                vec_t o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = (T)acc[i][j][4 * g + e];
                *reinterpret_cast<vec_t*>(slab + l31 * LDR + (j * 32 + g * 8 + hi * 4) * (int)sizeof(T)) = o;
            }
#pragma unroll
        for (int k = 0; k < 32 * LPR / 64; ++k) {
            const int row = k * (64 / LPR) + lane / LPR;
            const int64_t m = m0 + wm * 64 + i * 32 + row;
            typedef T slab_t __attribute__((ext_vector_type(E)));
            const slab_t s = *reinterpret_cast<const slab_t*>(slab + row * LDR + (lane % LPR) * 16);
            if (m < p.M && n < p.N) store_out<T, E>(C, ldc, m, n, p.N - n, s, OUT == 1 && p.accumulate);
        }
    }
#endif
}

// the splits' partial products together, in their order, + bias
template <typename T>
__global__ __launch_bounds__(256) void blocks_fold_kernel(const BlocksArgs p, int splits) {
    const int64_t n4 = (p.N + 3) / 4;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.M * n4; i += (int64_t)gridDim.x * 256) {
        const int64_t m = i / n4, n = i % n4 * 4, left = p.N - n;
        typedef float vec_t __attribute__((ext_vector_type(4), aligned(4)));
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (int z = 0; z < splits; ++z) {
            const float* c = p.part + ((int64_t)z * p.M + m) * p.N + n;
            if (left >= 4) s += *reinterpret_cast<const vec_t*>(c);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += e < left ? c[e] : 0.f;
        }
        T __attribute__((ext_vector_type(4))) o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)(s[e] + (p.bias && e < left ? p.bias[n + e] : 0.f));
        store_out<T, 4>((T*)p.C, p.ldc, m, n, left, o, p.accumulate != 0);
    }
}

struct BlocksPlan { int bn, splits, nk_split; };

// wide tiles where they alone fill the 256 CUs twice; otherwise narrow ones, and a long reduction is split until there are about 512 workgroups, at least eight
// blocks (16 steps) each
BlocksPlan blocks_plan(int64_t M, int64_t N, int64_t K) {
    const int64_t tm = (M + 127) / 128, nk = K / 128;
    if (N > 128 && tm * ((N + 255) / 256) >= 512) return {256, 1, (int)nk};
    const int64_t tiles = tm * ((N + 127) / 128);
    int64_t s = 512 / tiles;
    if (s > nk / 8) s = nk / 8;
    if (s < 2) return {128, 1, (int)nk};
    const int64_t per = ((nk + s - 1) / s + 3) / 4 * 4;
    return {128, (int)((nk + per - 1) / per), (int)per};
}

template <int FA, int BN>
void blocks_launch(const BlocksArgs& p, int splits, bool out_f32, hipStream_t s) {
    const dim3 grid(p.ntm * p.ntn, splits), block(256);
    if (splits > 1) {
        if constexpr (BN == 128) {
            const int64_t work = p.M * ((p.N + 3) / 4);
            const dim3 fold((unsigned)min((int64_t)4096, (work + 255) / 256));
            if (out_f32) {
                hipLaunchKernelGGL((blocks_gemm_kernel<FA, BN, 2, true>), grid, block, 0, s, p);
                hipLaunchKernelGGL((blocks_fold_kernel<float>), fold, block, 0, s, p, splits);
            } else {
                hipLaunchKernelGGL((blocks_gemm_kernel<FA, BN, 2, false>), grid, block, 0, s, p);
                hipLaunchKernelGGL((blocks_fold_kernel<bf16>), fold, block, 0, s, p, splits);
            }
        }
    } else if (out_f32) {
        hipLaunchKernelGGL((blocks_gemm_kernel<FA, BN, 1, true>), grid, block, 0, s, p);
    } else {
        hipLaunchKernelGGL((blocks_gemm_kernel<FA, BN, 0, false>), grid, block, 0, s, p);
    }
}

}  // namespace

extern "C" int64_t merlot_gemm_f8_blocks_workspace_bytes(int64_t M, int64_t N, int64_t K) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const BlocksPlan plan = blocks_plan(M, N, K);
    return plan.splits > 1 ? (int64_t)plan.splits * M * N * 4 : 0;
}

extern "C" int merlot_gemm_f8_blocks(const void* A8, int64_t lda, int fmt_a, const uint8_t* scale_a, int64_t ld_scale_a, const void* B8, int64_t ldb,
                                     const uint8_t* scale_b, int64_t ld_scale_b, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int out_f32,
                                     int accumulate, const float* bias, void* workspace, int64_t workspace_bytes, merlot_stream_t stream) {
    MERLOT_CHECK(A8 && B8 && scale_a && scale_b && C, MERLOT_ESHAPE, "merlot_gemm_f8_blocks: null operand");
    MERLOT_CHECK(M > 0 && N > 0 && K > 0 && K % 128 == 0 && K < ((int64_t)1 << 31), MERLOT_ESHAPE, "merlot_gemm_f8_blocks: bad size (K must be a multiple of 128)");
    MERLOT_CHECK(fmt_a == 0 || fmt_a == 1, MERLOT_EDTYPE, "merlot_gemm_f8_blocks: fmt_a must be 0 (e4m3) or 1 (e5m2)");
    MERLOT_CHECK(!accumulate || out_f32, MERLOT_EDTYPE, "merlot_gemm_f8_blocks: accumulation needs an fp32 output");
    MERLOT_CHECK(lda >= K && ldb >= K && ldc >= N && lda < (1 << 22) && ldb < (1 << 22), MERLOT_ESHAPE, "merlot_gemm_f8_blocks: bad leading dimension");
    MERLOT_CHECK(lda % 16 == 0 && ldb % 16 == 0 && (((uintptr_t)A8 | (uintptr_t)B8) & 15) == 0, MERLOT_EALIGN, "merlot_gemm_f8_blocks: operand rows must be 16-byte aligned");
    MERLOT_CHECK(ld_scale_a >= K / 128 && ld_scale_b >= K / 128 && ld_scale_a % 4 == 0 && ld_scale_b % 4 == 0 && ld_scale_a < (1 << 22) && ld_scale_b < (1 << 22) &&
                     (((uintptr_t)scale_a | (uintptr_t)scale_b) & 3) == 0,
                 MERLOT_EALIGN, "merlot_gemm_f8_blocks: scale rows must be 4-byte aligned and hold K / 128 bytes");
    const BlocksPlan plan = blocks_plan(M, N, K);
    MERLOT_CHECK(plan.splits == 1 || (workspace && workspace_bytes >= (int64_t)plan.splits * M * N * 4), MERLOT_ESHAPE, "merlot_gemm_f8_blocks: workspace too small");
    const int64_t ntm = (M + 127) / 128, ntn = (N + plan.bn - 1) / plan.bn;
    MERLOT_CHECK(ntm * ntn < ((int64_t)1 << 31), MERLOT_ESHAPE, "merlot_gemm_f8_blocks: too many tiles");
    const BlocksArgs p = {(const uint8_t*)A8, (const uint8_t*)B8, scale_a, scale_b, lda, ldb, ld_scale_a, ld_scale_b, C, ldc, bias, (float*)workspace, M, N,
                          (int)(K / 128), plan.nk_split, (int)ntm, (int)ntn, accumulate};
    hipStream_t s = (hipStream_t)stream;
    if (fmt_a == 0) {
        if (plan.bn == 256) blocks_launch<0, 256>(p, plan.splits, out_f32 != 0, s);
        else blocks_launch<0, 128>(p, plan.splits, out_f32 != 0, s);
    } else {
        if (plan.bn == 256) blocks_launch<1, 256>(p, plan.splits, out_f32 != 0, s);
        else blocks_launch<1, 128>(p, plan.splits, out_f32 != 0, s);
    }
    return merlot_launch_status("merlot_gemm_f8_blocks");
}
