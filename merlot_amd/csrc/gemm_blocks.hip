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
#include <utility>
#include "blocks8.h"

namespace {

struct BlocksArgs {
    const uint8_t *A, *B, *sa, *sb;
    int64_t lda, ldb, ldsa, ldsb;
    void* C; int64_t ldc;
    const float* bias;
    float* part;                             // split reductions: [splits][M][part_ld(N)] partial products
    int64_t M, N;
    int nk, nk_split, splits;                // blocks of 128 in all, per split
    int ntm, ntn;
    int accumulate;
    unsigned band_magic;                     // 2^32 / (4 ntn): blocks_wide_kernel
};

// rows of partial products start at multiples of 64 bytes, whatever N
__host__ __device__ __forceinline__ int64_t part_ld(int64_t N) { return (N + 15) & ~(int64_t)15; }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const uint8_t* p, int64_t row0, int64_t rows, int64_t ld, int64_t width) {
    // the rows of one tile as a buffer of their own: offsets stay small however large the operand is, and rows past its end read as zeros
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p + row0 * ld), 0, rows > 0 ? (int)((rows - 1) * ld + width) : 0, 0x00020000);
}

// up to E consecutive columns at c, `left` of which exist; add: onto what is there (fp32 only).  Outputs are stored past the caches (non-temporal): kept in the L2, a
// large output drives out the operands that the neighbouring tiles are about to read -- 101376 x 2304 x 768 takes 262 us that way and 194 us this way.
template <typename T, int E>
__device__ __forceinline__ void store_out(T* c, int64_t left, T __attribute__((ext_vector_type(E))) v, bool add) {
    typedef T vec_t __attribute__((ext_vector_type(E), aligned(sizeof(T))));
    if (left >= E) {
        if constexpr (sizeof(T) == 4)
            if (add) v += *reinterpret_cast<const vec_t*>(c);
        __builtin_nontemporal_store((vec_t)v, reinterpret_cast<vec_t*>(c));
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

// Tile 128 x BN, four waves (64 x 128 each for BN 256, 64 x 64 for BN 128), K-steps of 64, three step buffers filled by LDS-DMA two to three steps ahead, one
// barrier per step.  Two workgroups share a CU (72 + 6 KiB of LDS, 256 registers): while one waits, loads or stores its tile, the other multiplies.
// OUT: 0 bf16, 1 fp32, 2 fp32 partial products of a split reduction.  EXACT: through bf16 fragments (see above).
constexpr int direct_unroll(int mf) { return mf <= 2 ? 4 : 2; }       // blocks in flight per wave of blocks_direct_kernel
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
    auto issue = [&](int step, int base) {       // base: byte offset of the buffer
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            if (i < 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, LDS_PTR(lds + base + (wave * 2 + i) * 1024), 16, off[i], step * 64, 0, 0);
            else __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, LDS_PTR(lds + base + (8 + wave * (PIECES - 2) + i - 2) * 1024), 16, off[i], step * 64, 0, 0);
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
    auto fragment = [&](int base, unsigned row_off, unsigned c) -> i32x8 {
        const i32x4 x = *reinterpret_cast<const i32x4*>(lds + base + row_off + c * 16);
        const i32x4 y = *reinterpret_cast<const i32x4*>(lds + base + row_off + (c ^ 1) * 16);
        return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    // One step = two halves of the wave's columns.  The second half's B fragments are read while the first half multiplies, the NEXT step's A and first-half B
    // fragments while the second half does; the barrier stands between the halves: behind it the step's buffer is free (every read of it has returned) and takes
    // step t + 3, and step t + 1 is complete.
    const int steps = 2 * (kb1 - kb0);
    constexpr int NH = NJ / 2;
    issue(2 * kb0, 0);
    issue(2 * kb0 + 1, STEP);
    if (steps > 2) { issue(2 * kb0 + 2, 2 * STEP); wait_step<2 * PIECES>(); }
    else wait_step<PIECES>();
    __builtin_amdgcn_s_barrier();
    i32x8 fa[2][2], fb0[NH], fb1[NH];                    // fa: [parity of the step]
    int xa[2], xb[NJ];
    auto read_scales = [&](int w) {                      // a word holds four blocks' bytes
#pragma unroll
        for (int i = 0; i < 2; ++i) xa[i] = *reinterpret_cast<const int*>(scales + (wm * 64 + i * 32 + l31) * 16 + w * 4);
#pragma unroll
        for (int j = 0; j < NJ; ++j) xb[j] = *reinterpret_cast<const int*>(scales + (BM + wn * (BN / 2) + j * 32 + l31) * 16 + w * 4);
    };
    auto multiply = [&](const i32x8 (&a)[2], const i32x8 (&b)[NH], auto first) {
        constexpr int J0 = decltype(first)::value;
        if constexpr (!EXACT) {
#pragma unroll
            for (int j = 0; j < NH; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    acc[i][J0 + j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[j], a[i], acc[i][J0 + j], 0, FA, 0, xb[J0 + j], 0, xa[i]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {                // lane k-bytes 8 q ... : the same eight of both operands, which is all a dot product asks for
                bf16x8 wa[2], wb[NH];
#pragma unroll
                for (int i = 0; i < 2; ++i) wa[i] = widen<FA>(a[i][2 * q], a[i][2 * q + 1], scale_value(xa[i] & 255));
#pragma unroll
                for (int j = 0; j < NH; ++j) wb[j] = widen<0>(b[j][2 * q], b[j][2 * q + 1], scale_value(xb[J0 + j] & 255));
#pragma unroll
                for (int j = 0; j < NH; ++j)
#pragma unroll
                    for (int i = 0; i < 2; ++i) acc[i][J0 + j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[j], wa[i], acc[i][J0 + j], 0, 0, 0);
            }
        }
        // a use of the sums in this segment: without one the compiler sinks the (side-effect free) matrix instructions behind the reads they are meant to cover
#pragma unroll
        for (int j = 0; j < NH; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                f32x16& s = acc[i][J0 + j];
                asm volatile("" : "+v"(s));
            }
    };
    read_scales(0);
    int cur = 0;                                         // byte offset of step t's buffer
#pragma unroll
    for (int i = 0; i < 2; ++i) fa[0][i] = fragment(cur, ra_off[i], ca[i]);
#pragma unroll
    for (int j = 0; j < NH; ++j) fb0[j] = fragment(cur, rb_off[j], cb[j]);
    auto step = [&](int t, auto parity) {
        constexpr int P = decltype(parity)::value;
#pragma unroll
        for (int j = 0; j < NH; ++j) fb1[j] = fragment(cur, rb_off[NH + j], cb[NH + j]);
        __builtin_amdgcn_sched_barrier(0);
        multiply(fa[P], fb0, std::integral_constant<int, 0>{});
        __builtin_amdgcn_sched_barrier(0);
        // the last words of the old sixteen blocks were read eight steps ago, seven barriers back
        if (((t + 1) & (2 * SCALE_BLOCKS - 1)) == 0 && t + 1 < steps) load_scales(kb0 + ((t + 1) >> 1));
        if (t + 2 < steps) wait_step<PIECES>();
        else wait_step<0>();
        __builtin_amdgcn_s_barrier();
        if (t + 3 < steps) issue(2 * kb0 + t + 3, cur);
        cur = cur == 2 * STEP ? 0 : cur + STEP;
#pragma unroll
        for (int i = 0; i < 2; ++i) fa[P ^ 1][i] = fragment(cur, ra_off[i], ca[i]);      // (behind the last step: bytes nobody uses)
#pragma unroll
        for (int j = 0; j < NH; ++j) fb0[j] = fragment(cur, rb_off[j], cb[j]);
        __builtin_amdgcn_sched_barrier(0);
        multiply(fa[P], fb1, std::integral_constant<int, NH>{});
        __builtin_amdgcn_sched_barrier(0);
        if (P) {                                         // both steps of a block are done: the next byte
            if (((t + 1) & 7) == 0) {
                read_scales(((t + 1) >> 3) & 3);
            } else {
#pragma unroll
                for (int i = 0; i < 2; ++i) xa[i] = (int)((unsigned)xa[i] >> 8);
#pragma unroll
                for (int j = 0; j < NJ; ++j) xb[j] = (int)((unsigned)xb[j] >> 8);
            }
        }
    };
    for (int t = 0; t < steps; t += 2) {                 // (two steps per block: steps is even)
        step(t, std::integral_constant<int, 0>{});
        step(t + 1, std::integral_constant<int, 1>{});
    }
    // ---- epilogue: 32 rows at a time through a slab of the wave's own in the step buffers, so that memory sees whole rows of the wave's columns
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    typedef typename std::conditional<OUT == 0, bf16, float>::type T;
    constexpr int COLS = BN / 2, LDR = COLS * (int)sizeof(T) + 16, E = 16 / (int)sizeof(T), LPR = COLS / E;      // slab row in bytes; 16-byte groups per row
    static_assert(4 * 32 * LDR <= 3 * STEP, "slabs");
    uint8_t* const slab = lds + wave * 32 * LDR;
    const int64_t ldc = OUT == 2 ? part_ld(p.N) : p.ldc, n = n0 + wn * COLS + (lane % LPR) * E;
    T* const C = OUT == 2 ? (T*)p.part + (int64_t)blockIdx.y * p.M * ldc : (T*)p.C;
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
            if (m < p.M && n < p.N) store_out<T, E>(C + m * ldc + n, p.N - n, s, OUT == 1 && p.accumulate);
        }
    }
#endif
}

// Large outputs: 256 x 256 tiles, four waves of 128 x 128 -- ONE per SIMD, 256 accumulators each --, K-tiles of 128 (whole 128-byte lines per row, where 64-byte steps
// ask the L2 twice per line), two K-tile buffers.  A wave's next fragments are read, and the next K-tile is fetched, between its own matrix instructions; the one barrier
// per K-tile stands where the buffer's last reads have returned.  Persistent: workgroups walk the tiles of their XCD's band, the fetch stream runs on across tile ends, and
// a tile's stores drain while the next one multiplies.  fp32 outputs convert two fragment slices between every four matrix
// instructions, two conversions each (8192^3: 745 - 787 us = 1.4 - 1.5 PFLOP/s, the rate of a large bf16 product; 128 x 256 tiles 870).
constexpr int WIDE_BUF = 65536, WIDE_SCALES = 2 * WIDE_BUF, WIDE_BIAS = WIDE_SCALES + 512 * SCALE_BLOCKS, WIDE_SLAB = WIDE_BIAS + 2048;
constexpr int WIDE_LDS = WIDE_SLAB + 4 * 4096;           // two K-tiles, 16 blocks' scale bytes of 512 rows, two tiles' bias, a slab of 32 rows x 128 bytes per wave

template <typename F, int... U>
__device__ __forceinline__ void units(F& f, std::integer_sequence<int, U...>) { (f(std::integral_constant<int, U>{}), ...); }

// LINES: rows of C start at multiples of 64 bytes -- stored past the caches (a template: two branches with the same store would be merged into an ordinary one)
// OUT: 0 bf16, 1 fp32, 2 fp32 partial products of a split reduction; fp32 through bf16 fragments (the work items are (split, tile), split by split)
template <int FA, bool LINES, int OUT>
__global__ __launch_bounds__(256, 1) void blocks_wide_kernel(const BlocksArgs p) {
#ifdef __HIP_DEVICE_COMPILE__
    constexpr bool EXACT = OUT != 0;
    typedef typename std::conditional<EXACT, float, bf16>::type T;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hi = lane >> 5, l31 = lane & 31, wm = wave >> 1, wn = wave & 1;
    const int ntiles = p.ntm * p.ntn, nwg = gridDim.x;
    // XCD x's band of tiles, and this workgroup's walk through it
    const int items = OUT == 2 ? ntiles * p.splits : ntiles;
    const int xcd = (int)blockIdx.x & 7, q8 = items >> 3, r8 = items & 7;
    const int band = xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8, band_end = band + q8 + (xcd < r8 ? 1 : 0);
    const int stride = (nwg >> 3) + (xcd < (nwg & 7) ? 1 : 0);
    int tile = band + ((int)blockIdx.x >> 3);
    if (tile >= band_end) return;
    auto place = [&](int id, int& m0, int& n0) __attribute__((always_inline)) {         // bands of four tile rows, column by column (an XCD's 32 CUs: about 4 x 8 tiles)
        if constexpr (OUT == 2) id = (int)((unsigned)id % (unsigned)ntiles);
        const unsigned d = 4u * (unsigned)p.ntn;
        unsigned b = __umulhi((unsigned)id, p.band_magic), in = (unsigned)id - b * d;     // floor(2^32 / d): the quotient or one less
        if (in >= d) { ++b; in -= d; }
        const unsigned high = min(4u, (unsigned)p.ntm - b * 4u);
        const unsigned c = high == 4u ? in >> 2 : high == 3u ? __umulhi(in, 0x55555556u) : high == 2u ? in >> 1 : in;
        m0 = (int)(b * 4u + in - c * high) * 256;
        n0 = (int)c * 256;
    };
    auto first_of = [&](int id) __attribute__((always_inline)) -> int { return OUT == 2 ? (int)((unsigned)id / (unsigned)ntiles) * p.nk_split : 0; };
    auto count_of = [&](int first) __attribute__((always_inline)) -> int { return OUT == 2 ? min(p.nk_split, p.nk - first) : p.nk; };
    const int64_t K = (int64_t)p.nk * 128;
    // ---- fetch stream: 32 pieces of 8 rows x 128 bytes per operand and K-tile, 8 + 8 per wave.  Image: row r at r * 128, its 16-byte chunk c at c ^ ((r >> 1) & 7)
    unsigned offa[8], offb[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int row = (wave * 8 + i) * 8 + (lane >> 3);
        const unsigned ch = (unsigned)(((lane & 7) ^ (row >> 1)) & 7) * 16;
        offa[i] = (unsigned)(row * p.lda) + ch;
        offb[i] = (unsigned)(row * p.ldb) + ch;
    }
    __amdgpu_buffer_rsrc_t ra, rb;
    int s_tile = tile, s_kt = 0, s_end = p.nk;
    auto stream_to = [&](int id) __attribute__((always_inline)) {
        int m = 0, n = 0;
        s_kt = first_of(id);
        s_end = s_kt + count_of(s_kt);
        if (id < band_end) place(id, m, n);              // (behind the last tile: buffers without a byte -- the two K-tiles fetched ahead touch no memory)
        ra = rows_rsrc(p.A, m, id < band_end ? min((int64_t)256, p.M - m) : 0, p.lda, K);
        rb = rows_rsrc(p.B, n, id < band_end ? min((int64_t)256, p.N - n) : 0, p.ldb, K);
    };
    auto fetch_a = [&](int i, int buf) { __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, LDS_PTR(lds + buf + (wave * 8 + i) * 1024), 16, offa[i], s_kt * 128, 0, 0); };
    auto fetch_b = [&](int i, int buf) { __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, LDS_PTR(lds + buf + 32768 + (wave * 8 + i) * 1024), 16, offb[i], s_kt * 128, 0, 0); };
    auto advance = [&]() __attribute__((always_inline)) {                               // to the stream's next K-tile
        if (++s_kt == s_end) {
            s_tile += stride;
            stream_to(s_tile);
        }
    };
    // ---- scale words (16 blocks of 512 rows: eight words per thread) and bias, through registers into LDS
    int sw[8];
    float bias_reg;
    auto ask_scales = [&](int id, int kb) {              // kb: within the item
        int m, n;
        place(id, m, n);
        kb += first_of(id);
        const int64_t width = (p.nk + 3) & ~3;
        const __amdgpu_buffer_rsrc_t rsa = rows_rsrc(p.sa, m, min((int64_t)256, p.M - m), p.ldsa, width), rsb = rows_rsrc(p.sb, n, min((int64_t)256, p.N - n), p.ldsb, width);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const unsigned row = k * 64 + (tid >> 2), b = kb + (tid & 3) * 4;
            sw[k] = __builtin_amdgcn_raw_buffer_load_b32(rsa, row * (unsigned)p.ldsa + b, 0, 0);
            sw[4 + k] = __builtin_amdgcn_raw_buffer_load_b32(rsb, row * (unsigned)p.ldsb + b, 0, 0);
        }
    };
    auto put_scales = [&]() {
#pragma unroll
        for (int k = 0; k < 8; ++k) *reinterpret_cast<int*>(lds + WIDE_SCALES + (k * 64 + (tid >> 2)) * 16 + (tid & 3) * 4) = sw[k];
    };
    auto ask_bias = [&](int id) {
        int m, n;
        place(id, m, n);
        bias_reg = p.bias && n + tid < p.N ? p.bias[n + tid] : 0.f;
    };
    // ---- fragments
    const unsigned fra = (unsigned)(wm * 128 + l31) * 128, frb = 32768u + (unsigned)(wn * 128 + l31) * 128;     // + 32 rows = 4 096 bytes each, same exchange
    const unsigned fx = (unsigned)(l31 >> 1) & 7;
    auto chunk = [&](unsigned base, int k2, int part) -> i32x4 {           // half a fragment: 16 bytes of a row
        return *reinterpret_cast<const i32x4*>(lds + base + (((unsigned)(4 * k2 + 2 * hi + part) ^ fx) & 7) * 16);
    };
    auto whole = [](const i32x4 (&f)[2]) -> i32x8 { return __builtin_shufflevector(f[0], f[1], 0, 1, 2, 3, 4, 5, 6, 7); };
    int xa[4], xb[4];
    auto read_scales = [&](int w) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            xa[i] = *reinterpret_cast<const int*>(lds + WIDE_SCALES + (wm * 128 + i * 32 + l31) * 16 + w * 4);
            xb[i] = *reinterpret_cast<const int*>(lds + WIDE_SCALES + (256 + wn * 128 + i * 32 + l31) * 16 + w * 4);
        }
    };
    f32x16 acc[4][4];
    f32x16 zero;
#pragma unroll
    for (int r = 0; r < 16; ++r) zero[r] = 0.f;
    i32x4 fa[2][4][2], fb[2][4][2];                      // [half K-tile][32 rows][16 bytes]
    // chunk f (0 ... 15) of the fragments of half H in the order the products ask for them: B 0, A 0, A 1, A 2, A 3, B 1, B 2, B 3
    auto read_chunk = [&](auto hc, int f, unsigned base) __attribute__((always_inline)) {
        constexpr int H = decltype(hc)::value;
        // (fp32: the first halves of all fragments, which are converted first, then the others)
        const int k = EXACT ? f & 7 : f >> 1, part = EXACT ? f >> 3 : f & 1;
        if (k == 0 || k >= 5) { const int j = k == 0 ? 0 : k - 4; fb[H][j][part] = chunk(base + frb + j * 4096, H, part); }
        else fa[H][k - 1][part] = chunk(base + fra + (k - 1) * 4096, H, part);
    };
    // fp32: slice q (16 of the half K-tile's 64, eight per half wave) of the fragments as bf16, the scale included; the next slice is converted between the products
    bf16x8 wa[2][4], wb[2][4];                           // [parity of the slice]
    float va[4], vb[4];                                  // the block's scales
    auto scale_floats = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            va[i] = scale_value(xa[i] & 255);
            vb[i] = scale_value(xb[i] & 255);
        }
    };
    auto convert = [&](auto hc, int q, int f) __attribute__((always_inline)) {       // f: 0 ... 3 rows of A, 4 ... 7 of B
        constexpr int H = decltype(hc)::value;
        if (f < 4) wa[q & 1][f] = widen<FA>(fa[H][f][q >> 1][2 * (q & 1)], fa[H][f][q >> 1][2 * (q & 1) + 1], va[f]);
        else wb[q & 1][f - 4] = widen<0>(fb[H][f - 4][q >> 1][2 * (q & 1)], fb[H][f - 4][q >> 1][2 * (q & 1) + 1], vb[f - 4]);
    };
    // one half K-tile: the products with the fragments of half P; between them the other half's fragments are read from the buffer at `next`, and with FETCH the stream's
    // K-tile is fetched into the one at `into`
    auto half = [&](auto pc, auto firstc, auto fetchc, unsigned next, int into) __attribute__((always_inline)) {
        constexpr int P = decltype(pc)::value;
        constexpr bool FIRST = decltype(firstc)::value, FETCH = decltype(fetchc)::value;
        if constexpr (EXACT && P == 0) {
            scale_floats();
#pragma unroll
            for (int f = 0; f < 8; ++f) convert(pc, 0, f);
        }
        // sixteen slots of one matrix instruction (64 cycles; fp32: 128): one read and one fetch in half 1; in half 0 two reads in each of the first eight, so that they have returned
        // where the barrier behind the half asks for it
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int i = k & 3, j = k >> 2;
            if (P == 1) {
                read_chunk(std::integral_constant<int, P ^ 1>{}, k, next);
            } else if (k < 8) {
                read_chunk(std::integral_constant<int, P ^ 1>{}, 2 * k, next);
                read_chunk(std::integral_constant<int, P ^ 1>{}, 2 * k + 1, next);
            }
            if constexpr (FETCH) {
                if (k & 1) fetch_b(k >> 1, into);
                else fetch_a(k >> 1, into);
            }
            if constexpr (!EXACT) {
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(whole(fb[P][j]), whole(fa[P][i]), FIRST ? zero : acc[i][j], 0, FA, 0, xb[j], 0, xa[i]);
            } else {                                     // a slot: column j of slice q = k / 4, four matrix instructions of 32 cycles
                const int q = k >> 2, c = k & 3;
                // the next slice's fragments, two a slot; behind half 0 those of half 1 (half 0's own first slice waits for its block's scales)
                if (q < 3) {
                    convert(pc, q + 1, 2 * c);
                    convert(pc, q + 1, 2 * c + 1);
                } else if (P == 0) {
                    convert(std::integral_constant<int, 1>{}, 0, 2 * c);
                    convert(std::integral_constant<int, 1>{}, 0, 2 * c + 1);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc[r][c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wb[q & 1][c], wa[q & 1][r], FIRST && q == 0 ? zero : acc[r][c], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) {                // (a use in this segment: see blocks_gemm_kernel; the 256 sums fill the accumulation registers)
                f32x16& s = acc[i][j];
                asm volatile("" : "+a"(s));
            }
        __builtin_amdgcn_sched_barrier(0);
    };
    typedef std::integral_constant<int, 0> c0_t;
    typedef std::integral_constant<int, 1> c1_t;
    typedef std::integral_constant<bool, false> no_t;
    typedef std::integral_constant<bool, true> yes_t;

    // ---- prologue
    ask_scales(tile, 0);
    ask_bias(tile);
    put_scales();
    *reinterpret_cast<float*>(lds + WIDE_BIAS + tid * 4) = bias_reg;
    stream_to(tile);
#pragma unroll
    for (int b = 0; b < 2; ++b) {                        // K-tiles 0 and 1 (the host launches this kernel for K >= 256 only)
#pragma unroll
        for (int i = 0; i < 8; ++i) { fetch_a(i, b * WIDE_BUF); fetch_b(i, b * WIDE_BUF); }
        advance();
    }
    wait_step<16>();
    __builtin_amdgcn_s_barrier();
    unsigned buf = 0;
#pragma unroll
    for (int f = 0; f < 16; ++f) read_chunk(c0_t{}, f, buf);
    int bias_at = WIDE_BIAS, stores = 0;                 // stores: this wave's stores behind the newest fetch, at least
    while (true) {
        int m0, n0;
        place(tile, m0, n0);
        const int next_tile = tile + stride;
        const bool last = next_tile >= band_end;
        const int kb0 = first_of(tile), nk = count_of(kb0);          // the item's blocks
        read_scales(0);
        auto ktile = [&](int kt, auto firstc) __attribute__((always_inline)) {
            half(c0_t{}, firstc, no_t{}, buf, 0);
            // K-tile kt + 1 has to be complete, and everybody's reads of this buffer (lgkmcnt: ours) done; behind the first K-tile's fetches only the last tile's stores
            // are younger
            if (decltype(firstc)::value && stores >= 32) wait_step<32>();
            else wait_step<0>();
            __builtin_amdgcn_s_barrier();
            half(c1_t{}, no_t{}, yes_t{}, buf ^ WIDE_BUF, (int)buf);
            advance();
            buf ^= WIDE_BUF;
            if (((kt + 1) & 15) == 0 && kt + 1 < nk) {   // the next sixteen blocks' bytes (the old ones' last words were read three K-tiles ago)
                ask_scales(tile, kt + 1);
                put_scales();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
            }
            if (((kt + 1) & 3) == 0) {
                if (kt + 1 < nk) read_scales(((kt + 1) >> 2) & 3);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    xa[i] = (int)((unsigned)xa[i] >> 8);
                    xb[i] = (int)((unsigned)xb[i] >> 8);
                }
            }
        };
        ktile(0, yes_t{});
        for (int kt = 1; kt < nk; ++kt) ktile(kt, no_t{});
        if (!last) {
            ask_scales(next_tile, 0);
            ask_bias(next_tile);
        } else {
            wait_step<0>();                              // the fetches ahead (zeros, from buffers without a byte) have left the LDS before the workgroup does
        }
        // ---- epilogue: units of 32 rows x 64 columns (fp32: 32) through the wave's slab (16-byte chunk c of row r at c ^ (r & 7)).  Unit u + 1 is rounded while unit u's writes and reads
        // travel, and unit u is stored behind that: nothing waits for the slab.
        uint8_t* const slab = lds + WIDE_SLAB + wave * 4096;
        int el = lane;                                   // the epilogue's addresses are made here, tile by tile: hoisted out of the tile loop they would fill the registers
        asm volatile("" : "+v"(el));
        const int e31 = el & 31, eh = el >> 5;
        const bool inside = m0 + 256 <= p.M && n0 + 256 <= p.N;
        constexpr int E = 16 / (int)sizeof(T), UC = 8 * E;           // values per lane, columns per unit
        const int64_t row0 = m0 + wm * 128 + (el >> 3), col0 = n0 + wn * 128 + (el & 7) * E;
        const int m_left = (int)max((int64_t)-1, min(p.M - row0, (int64_t)256)), n_left = (int)max((int64_t)-1, min(p.N - col0, (int64_t)256));
        const int64_t ldc = OUT == 2 ? part_ld(p.N) : p.ldc;
        T* out = (OUT == 2 ? (T*)p.part + (int64_t)(kb0 / p.nk_split) * p.M * ldc : (T*)p.C) + row0 * ldc + col0;    // this lane's piece of the slab's rows 0 ... 7
        typedef T __attribute__((ext_vector_type(4))) quad_t;
        typedef T __attribute__((ext_vector_type(E))) piece_t;
        constexpr int Q = UC / 8;                        // quads of a lane (its row, every eighth group of four columns)
        quad_t o[Q];
        piece_t v[4];
        f32x4 bias[Q];                                   // of the unit's columns
        auto ask = [&](int block) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < Q; ++k)
                if constexpr (OUT != 2) bias[k] = *reinterpret_cast<const f32x4*>(lds + bias_at + (wn * 128 + block * UC + k * 8 + eh * 4) * 4);
                else bias[k] = f32x4{0.f, 0.f, 0.f, 0.f};
        };
        auto round = [&](auto uc) __attribute__((always_inline)) {
            constexpr int U = decltype(uc)::value, I = U & 3, J = (U >> 2) * (UC / 32);   // column blocks outside: each one's bias is read once
            f32x16 &s0 = acc[I][J], &s1 = acc[I][EXACT ? J : J + 1];
            asm volatile("" : "+a"(s0));                 // fetched from the accumulation registers here, not all sums at the loop's end
            if constexpr (!EXACT) asm volatile("" : "+a"(s1));
#pragma unroll
            for (int k = 0; k < Q; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[k][e] = (T)((k < 4 ? s0 : s1)[4 * (k & 3) + e] + bias[k][e]);
        };
        auto write = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < Q; ++k)
                if constexpr (EXACT) *reinterpret_cast<quad_t*>(slab + e31 * 128 + ((((2 * k + eh) ^ e31) & 7) << 4)) = o[k];
                else *reinterpret_cast<quad_t*>(slab + e31 * 128 + (((k ^ e31) & 7) << 4) + eh * 8) = o[k];
        };
        auto read = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const piece_t*>(slab + (k * 8 + (el >> 3)) * 128 + (((el ^ (el >> 3)) & 7) << 4));
        };
        auto store = [&](auto uc) __attribute__((always_inline)) {
            constexpr int U = decltype(uc)::value, I = U & 3, C0 = (U >> 2) * UC;
            typedef T out_t __attribute__((ext_vector_type(E), aligned(sizeof(T))));
            if (inside) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    out_t* c = reinterpret_cast<out_t*>(out + (I * 32 + k * 8) * ldc + C0);
                    if constexpr (LINES) __builtin_nontemporal_store((out_t)v[k], c);
                    else *c = v[k];
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (I * 32 + k * 8 < m_left && C0 < n_left) store_out<T, E>(out + (I * 32 + k * 8) * ldc + C0, n_left - C0, v[k], false);
            }
        };
        auto unit = [&](auto uc) __attribute__((always_inline)) {
            constexpr int U = decltype(uc)::value;
            if constexpr ((U & 3) == 0) ask(U >> 2);
            round(uc);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (U > 0) store(std::integral_constant<int, U - 1>{});
            write();
            __builtin_amdgcn_sched_barrier(0);
            read();                                      // (LDS operations of a wave keep their order)
        };
        units(unit, std::make_integer_sequence<int, 4 * (128 / UC)>{});
        store(std::integral_constant<int, 4 * (128 / UC) - 1>{});
        if (last) break;
        stores = inside ? 16 * (128 / UC) : 0;
        tile = next_tile;
        put_scales();                                    // every wave is behind its last read of the old words (a barrier per K-tile)
        bias_at = bias_at == WIDE_BIAS ? WIDE_BIAS + 1024 : WIDE_BIAS;
        *reinterpret_cast<float*>(lds + bias_at + tid * 4) = bias_reg;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
    }
#endif
}

// Few rows, or little work: 16 NF columns x 16 MF rows per workgroup, the reduction dealt out block by block to its eight waves and joined once, in wave order, through
// LDS.  The operands go straight from memory to the registers (16 rows x 128 bytes: whole lines), every load of UNROLL blocks in flight at once: what bounds such a
// product is one round trip to memory, and the operands' way through the L2.
template <int FA, int MF, int NF, typename T>
__global__ __launch_bounds__(512) void blocks_direct_kernel(const BlocksArgs p) {
#ifdef __HIP_DEVICE_COMPILE__
    constexpr bool EXACT = sizeof(T) == 4;
    constexpr int UNROLL = direct_unroll(MF);
    __shared__ f32x4 part[8][MF * NF][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l15 = lane & 15, quarter = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NF), m0 = (int64_t)blockIdx.y * (16 * MF);
    const int64_t K = (int64_t)p.nk * 128;
    const int rows_a = (int)min((int64_t)(16 * MF), p.M - m0), rows_b = (int)min((int64_t)(16 * NF), p.N - n0);
    const __amdgpu_buffer_rsrc_t ra = rows_rsrc(p.A, m0, rows_a, p.lda, K), rb = rows_rsrc(p.B, n0, rows_b, p.ldb, K);
    const __amdgpu_buffer_rsrc_t rsa = rows_rsrc(p.sa, m0, rows_a, p.ldsa, p.nk), rsb = rows_rsrc(p.sb, n0, rows_b, p.ldsb, p.nk);
    f32x4 acc[MF][NF];
#pragma unroll
    for (int f = 0; f < MF; ++f)
#pragma unroll
        for (int g = 0; g < NF; ++g) acc[f][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    const unsigned oa = (unsigned)(l15 * p.lda) + quarter * 32, ob = (unsigned)(l15 * p.ldb) + quarter * 32, osa = (unsigned)(l15 * p.ldsa), osb = (unsigned)(l15 * p.ldsb);
    for (int kb = wave; kb < p.nk; kb += 8 * UNROLL) {
        i32x4 a[UNROLL][MF][2], b[UNROLL][NF][2];
        int xa[UNROLL][MF], xb[UNROLL][NF];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int k = kb + 8 * u;                    // (blocks past the last one: zeros times 2^0, without a trip to memory)
            const bool there = k < p.nk;
#pragma unroll
            for (int g = 0; g < NF; ++g) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    b[u][g][h] = there ? __builtin_amdgcn_raw_buffer_load_b128(rb, ob + (unsigned)(g * 16 * p.ldb) + h * 16, k * 128, 0) : i32x4{0, 0, 0, 0};
                xb[u][g] = there ? __builtin_amdgcn_raw_buffer_load_b8(rsb, osb + (unsigned)(g * 16 * p.ldsb), k, 0) : 127;
            }
#pragma unroll
            for (int f = 0; f < MF; ++f) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    a[u][f][h] = there ? __builtin_amdgcn_raw_buffer_load_b128(ra, oa + (unsigned)(f * 16 * p.lda) + h * 16, k * 128, 0) : i32x4{0, 0, 0, 0};
                xa[u][f] = there ? __builtin_amdgcn_raw_buffer_load_b8(rsa, osa + (unsigned)(f * 16 * p.ldsa), k, 0) : 127;
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if constexpr (!EXACT) {
#pragma unroll
                for (int f = 0; f < MF; ++f)
#pragma unroll
                    for (int g = 0; g < NF; ++g)
                        acc[f][g] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(b[u][g][0], b[u][g][1], 0, 1, 2, 3, 4, 5, 6, 7),
                                                                                     __builtin_shufflevector(a[u][f][0], a[u][f][1], 0, 1, 2, 3, 4, 5, 6, 7), acc[f][g], 0, FA, 0,
                                                                                     xb[u][g], 0, xa[u][f]);
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    bf16x8 wb[NF];
#pragma unroll
                    for (int g = 0; g < NF; ++g) wb[g] = widen<0>(b[u][g][q >> 1][2 * (q & 1)], b[u][g][q >> 1][2 * (q & 1) + 1], scale_value(xb[u][g] & 255));
#pragma unroll
                    for (int f = 0; f < MF; ++f) {
                        const bf16x8 wa = widen<FA>(a[u][f][q >> 1][2 * (q & 1)], a[u][f][q >> 1][2 * (q & 1) + 1], scale_value(xa[u][f] & 255));
#pragma unroll
                        for (int g = 0; g < NF; ++g) acc[f][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb[g], wa, acc[f][g], 0, 0, 0);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int f = 0; f < MF; ++f)
#pragma unroll
        for (int g = 0; g < NF; ++g) part[wave][f * NF + g][lane] = acc[f][g];
    __syncthreads();
    // lane <-> row (lane & 15) of A, register r <-> column 4 (lane >> 4) + r
    if (wave < MF * NF) {
        f32x4 s = part[0][wave][lane];
#pragma unroll
        for (int w = 1; w < 8; ++w) s += part[w][wave][lane];
        const int64_t m = m0 + wave / NF * 16 + l15, n = n0 + wave % NF * 16 + quarter * 4, left = p.N - n;
        if (m < p.M && left > 0) {
            T __attribute__((ext_vector_type(4))) o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (T)(s[e] + (p.bias && e < left ? p.bias[n + e] : 0.f));
            store_out<T, 4>((T*)p.C + m * p.ldc + n, left, o, p.accumulate != 0);
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
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (int z = 0; z < splits; ++z) {
            const f32x4 c = *reinterpret_cast<const f32x4*>(p.part + ((int64_t)z * p.M + m) * part_ld(p.N) + n);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += e < left ? c[e] : 0.f;
        }
        T __attribute__((ext_vector_type(4))) o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (T)(s[e] + (p.bias && e < left ? p.bias[n + e] : 0.f));
        store_out<T, 4>((T*)p.C + m * p.ldc + n, left, o, p.accumulate != 0);
    }
}

struct BlocksPlan { int bm, bn, splits, nk_split; };

// Straight from memory where every wave has its whole share of the reduction in flight at once (twice at most, with 16 rows) and the operands' way through the L2 --
// workgroups x (rows + columns) each -- stays short (us, 128-row tiles : direct): 1 x 2304 x 768 6.8 : 3.0, 32 x 4096 x 4096 12.1 : 10.8, 700 x 500 x 1024 9.3 : 6.5,
// 512 x 1024 x 1024 8.5 : 6.2, 100 x 4096 x 2048 12.1 : 9.7; but 16 x 50370 x 768 10.9 : 17.1, 64 x 4096 x 4096 13.3 : 19.3, 1000 x 1000 x 1024 9.0 : 11.1.
// bf16 outputs take 256 x 256 tiles where those fill the 256 CUs and the reduction is long enough to pay for an epilogue nobody covers (us, 128 x 256 tiles : 256 x 256):
//   101376 x 2304 x 384 139 : 138, x 512 161 : 139, x 768 224 : 200; 65536 x 768 x 768 55 : 49; 32768 x 4096 x 1024 159 : 142; 8192^3 513 : 400
// With rows of C that start inside a 64-byte sector their 128-byte row pieces are written as parts of lines, past the caches or not: 101376 x 2296 x 768 225 : 306, and only a
// long reduction hides it (30000 x 2296 x 2048 163 : 147, x 4096 297 : 254; 4099 x 50370 x 2048 467 : 476).
// fp32 outputs with such rows: 16384 x 4096 x 256 70 : 67, x 768 118 : 112; 8192^3 870 : 787; 4099 x 50304 x 768 344 : 322; with others not (4099 x 50370 x 768 374 : 458).  Added
// onto what is there they stay with 128 x 256 (the wide epilogue has no time to wait for old values).  Their long reductions are split over 256 x 256 tiles, at least half of which is
// the product's, where a workgroup gets ten blocks, or 18 if narrow tiles need no split (split over narrow tiles : 256 x 256): 4096 x 1024 x 32768 235 : 209, 2304 x 768 x 101376
// 325 : 288, x 12544 65 : 60, 2304 x 2304 x 8192 99 : 92; but 1024 x 1024 x 16384 46 : 52, 1000 x 4096 x 4096 43 : 55, 64 x 8192 x 8192 28 : 39.
// 128 x 256 where those fill the CUs twice; otherwise the reduction is split, or narrow tiles.
BlocksPlan blocks_plan(int64_t M, int64_t N, int64_t K, bool out_bf16, bool accumulate, bool whole_lines) {
    const int64_t tm = (M + 127) / 128, nk = K / 128;
    // straight from memory: 16 x 16, 32 x 16 or 64 x 32 outputs per workgroup
    const int mf = M <= 16 ? 1 : M <= 32 ? 2 : 4, nf = mf == 4 ? 2 : 1;
    if (nk <= 8 * direct_unroll(mf) * (mf == 1 ? 2 : 1) && (M + 16 * mf - 1) / (16 * mf) * ((N + 16 * nf - 1) / (16 * nf)) * (mf + nf) <= 3000) return {16 * mf, 16 * nf, 1, (int)nk};
    const int64_t tw = ((M + 255) / 256) * ((N + 255) / 256), wide = tm * ((N + 255) / 256), narrow = tm * ((N + 127) / 128);     // tiles of 256 x 256, 128 x 256, 128 x 128
    if (out_bf16 && nk >= (whole_lines ? 4 : 16) && tw >= 256) return {256, 256, 1, (int)nk};
    if (!out_bf16 && !accumulate && whole_lines && nk >= 2 && tw >= 256) return {256, 256, 1, (int)nk};
    if (!out_bf16 && tw <= 128 && 2 * M * N >= tw * 65536 && nk * tw / 256 >= (narrow > 128 ? 18 : 10)) {
        const int64_t s = 256 / tw, per = ((nk + s - 1) / s + 3) / 4 * 4;
        if ((nk + per - 1) / per > 1) return {256, 256, (int)((nk + per - 1) / per), (int)per};
    }
    if (N > 128 && wide >= 512) return {128, 256, 1, (int)nk};
    // long reductions are split: 128 x 256 tiles over three quarters of both places of every CU at least, where each workgroup keeps 24 blocks (us, bf16, narrow tiles in 7 parts : this way:
    // 2304 x 768 x 101376 280 : 238, x 24576 76 : 68; with 378 workgroups, 768 x 768 x 65536, 67 : 83); otherwise narrow tiles over one place of every CU, six blocks each at least (a
    // second workgroup on a CU gains 8 % of the time per block and costs another set of partial products: 1024 x 1024 x 8192, 64 tiles, in 4 : 8 parts 22 : 27, 256 x 4096 x 4096
    // 18 : 22).  Up to 16 blocks the second launch costs more than it saves (1024 x 1024 x 2048 whole 13, in two 15; 2000 x 1000 x 2048 14 : 19).
    auto parts = [&](int bn, int64_t s) -> BlocksPlan {
        const int64_t per = ((nk + s - 1) / s + 3) / 4 * 4;
        return {128, bn, (int)((nk + per - 1) / per), (int)per};
    };
    const int64_t sw = min(512 / wide, nk / 24), sn = min(256 / narrow, nk / 6);
    if (N > 128 && narrow <= 256 && sw >= 2 && wide * sw >= 384) return parts(256, sw);
    if (nk > 16 && sn >= 2) return parts(128, sn);
    return {128, 128, 1, (int)nk};
}

template <typename T>
void blocks_fold_launch(const BlocksArgs& p, hipStream_t s) {
    const int64_t work = p.M * ((p.N + 3) / 4);
    hipLaunchKernelGGL((blocks_fold_kernel<T>), dim3((unsigned)min((int64_t)4096, (work + 255) / 256)), dim3(256), 0, s, p, p.splits);
}

template <int FA, bool LINES, int OUT>
int blocks_wide_launch(const BlocksArgs& p, hipStream_t s) {
    const int items = p.ntm * p.ntn * p.splits;
    MERLOT_ENSURE_LDS((blocks_wide_kernel<FA, LINES, OUT>), WIDE_LDS, "merlot_gemm_f8_blocks");
    hipLaunchKernelGGL((blocks_wide_kernel<FA, LINES, OUT>), dim3(items < 256 ? items : 256), dim3(256), WIDE_LDS, s, p);
    if (OUT == 2) blocks_fold_launch<float>(p, s);
    return MERLOT_OK;
}

template <int FA>
int blocks_wide(const BlocksArgs& p, bool out_f32, bool lines, hipStream_t s) {
    if (p.splits > 1) return blocks_wide_launch<FA, true, 2>(p, s);
    if (out_f32) return blocks_wide_launch<FA, true, 1>(p, s);
    return lines ? blocks_wide_launch<FA, true, 0>(p, s) : blocks_wide_launch<FA, false, 0>(p, s);
}

template <int FA, typename T>
void blocks_direct_launch(const BlocksArgs& p, int bm, hipStream_t s) {
    const dim3 grid(p.ntn, p.ntm), block(512);
    if (bm == 16) hipLaunchKernelGGL((blocks_direct_kernel<FA, 1, 1, T>), grid, block, 0, s, p);
    else if (bm == 32) hipLaunchKernelGGL((blocks_direct_kernel<FA, 2, 1, T>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((blocks_direct_kernel<FA, 4, 2, T>), grid, block, 0, s, p);
}

template <int FA, int BN>
void blocks_launch(const BlocksArgs& p, bool out_f32, hipStream_t s) {
    const dim3 grid(p.ntm * p.ntn, p.splits), block(256);
    if (p.splits > 1) {
        if (out_f32) {
            hipLaunchKernelGGL((blocks_gemm_kernel<FA, BN, 2, true>), grid, block, 0, s, p);
            blocks_fold_launch<float>(p, s);
        } else {
            hipLaunchKernelGGL((blocks_gemm_kernel<FA, BN, 2, false>), grid, block, 0, s, p);
            blocks_fold_launch<bf16>(p, s);
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
    int splits = 1;                                      // whatever the output's type and alignment
    for (int k = 0; k < 8; ++k) splits = max(splits, blocks_plan(M, N, K, k & 1, k & 2, k & 4).splits);
    return splits > 1 ? (int64_t)splits * M * part_ld(N) * 4 : 0;
}

extern "C" int merlot_gemm_f8_blocks(const void* A8, int64_t lda, int fmt_a, const uint8_t* scale_a, int64_t ld_scale_a, const void* B8, int64_t ldb,
                                     const uint8_t* scale_b, int64_t ld_scale_b, void* C, int64_t ldc, int64_t M, int64_t N, int64_t K, int out_f32,
                                     int accumulate, const float* bias, void* workspace, int64_t workspace_bytes, merlot_stream_t stream) {
    MERLOT_CHECK(A8 && B8 && scale_a && scale_b && C, MERLOT_ESHAPE, "merlot_gemm_f8_blocks: null operand");
    MERLOT_CHECK(M > 0 && N > 0 && K > 0 && K % 128 == 0 && M < ((int64_t)1 << 31) - 256 && N < ((int64_t)1 << 31) - 256, MERLOT_ESHAPE,
                 "merlot_gemm_f8_blocks: bad size (K must be a multiple of 128)");
    MERLOT_CHECK(fmt_a == 0 || fmt_a == 1, MERLOT_EDTYPE, "merlot_gemm_f8_blocks: fmt_a must be 0 (e4m3) or 1 (e5m2)");
    MERLOT_CHECK(!accumulate || out_f32, MERLOT_EDTYPE, "merlot_gemm_f8_blocks: accumulation needs an fp32 output");
    MERLOT_CHECK(lda >= K && ldb >= K && ldc >= N && lda < (1 << 22) && ldb < (1 << 22), MERLOT_ESHAPE, "merlot_gemm_f8_blocks: bad leading dimension");
    MERLOT_CHECK(lda % 16 == 0 && ldb % 16 == 0 && (((uintptr_t)A8 | (uintptr_t)B8) & 15) == 0, MERLOT_EALIGN, "merlot_gemm_f8_blocks: operand rows must be 16-byte aligned");
    MERLOT_CHECK(ld_scale_a >= K / 128 && ld_scale_b >= K / 128 && ld_scale_a % 4 == 0 && ld_scale_b % 4 == 0 && ld_scale_a < (1 << 22) && ld_scale_b < (1 << 22) &&
                     (((uintptr_t)scale_a | (uintptr_t)scale_b) & 3) == 0,
                 MERLOT_EALIGN, "merlot_gemm_f8_blocks: scale rows must be 4-byte aligned and hold K / 128 bytes");
    const bool whole_lines = (((uintptr_t)C | (uint64_t)ldc * (out_f32 ? 4 : 2)) & 63) == 0;
    const BlocksPlan plan = blocks_plan(M, N, K, !out_f32, accumulate != 0, whole_lines);
    MERLOT_CHECK(plan.splits == 1 || (workspace && workspace_bytes >= (int64_t)plan.splits * M * part_ld(N) * 4 && ((uintptr_t)workspace & 15) == 0), MERLOT_ESHAPE, "merlot_gemm_f8_blocks: workspace too small, or not 16-byte aligned");
    const int64_t ntm = (M + plan.bm - 1) / plan.bm, ntn = (N + plan.bn - 1) / plan.bn;
    MERLOT_CHECK(ntm * ntn < ((int64_t)1 << 24), MERLOT_ESHAPE, "merlot_gemm_f8_blocks: too many tiles");
    const BlocksArgs p = {(const uint8_t*)A8, (const uint8_t*)B8, scale_a, scale_b, lda, ldb, ld_scale_a, ld_scale_b, C, ldc, bias, (float*)workspace, M, N,
                          (int)(K / 128), plan.nk_split, plan.splits, (int)ntm, (int)ntn, accumulate, (unsigned)(((uint64_t)1 << 32) / (4 * (uint64_t)ntn))};
    hipStream_t s = (hipStream_t)stream;
    if (plan.bn <= 64) {
        if (out_f32) fmt_a == 0 ? blocks_direct_launch<0, float>(p, plan.bm, s) : blocks_direct_launch<1, float>(p, plan.bm, s);
        else fmt_a == 0 ? blocks_direct_launch<0, bf16>(p, plan.bm, s) : blocks_direct_launch<1, bf16>(p, plan.bm, s);
    } else if (plan.bm == 256) {
        const int rc = fmt_a == 0 ? blocks_wide<0>(p, out_f32 != 0, whole_lines, s) : blocks_wide<1>(p, out_f32 != 0, whole_lines, s);
        if (rc != MERLOT_OK) return rc;
    } else if (fmt_a == 0) {
        if (plan.bn == 256) blocks_launch<0, 256>(p, out_f32 != 0, s);
        else blocks_launch<0, 128>(p, out_f32 != 0, s);
    } else {
        if (plan.bn == 256) blocks_launch<1, 256>(p, out_f32 != 0, s);
        else blocks_launch<1, 128>(p, out_f32 != 0, s);
    }
    return merlot_launch_status("merlot_gemm_f8_blocks");
}
