// Products of a few 16-bit rows with a matrix of 4-bit weights: y[m, n] = sum_k x[m, k] W[n, k], m <= 64.
//
//   MX fp4   W = e2m1(code) 2^(byte - 127), one scale byte per 32 k: the weights of the MX fp4 GEMM, byte for byte
//   int4     W = s (code - z), code 0 .. 15, one 16-bit s (and z; 8 without) per group of 32, 64 or 128 k
// two codes a byte, the lower k in the low nibble.  The sum of 32 k is taken on the codes, exactly representable in
// float16, by the tensor core with fp32 accumulation, and scaled afterwards:
//   y += 2^E s (sum (code) x' - z sum x'),   x = 2^E x'
// x' is x in float16.  float16 rows go in as they are (E = 0).  bfloat16 rows have float16's precision and more range,
// so each run of 256 gets the power of two that brings its largest element into [2^14, 2^15): every element down to
// 2^-31 of the largest keeps all its bits, below that the error is at most 2^-40 of the largest, far under the
// rounding of the fp32 sum.  Weights go through float16 because one conversion instruction turns two e2m1 codes into a
// float16 pair, and an int4 code is the float16 subnormal code * 2^-24 after one mask; to bfloat16 both take three to
// four half-rate integer operations a pair.
//
// Bound by HBM: n k / 2 bytes of weights are read once, everything else is small.  Weights are the 16-row operand of
// mma.m16n8k16, the rows of x its eight columns; the order of k inside 32 is free as long as both operands agree: lane t
// of a quad takes k = 8t .. 8t + 7 (one word of codes).  The rows of W are dealt out evenly, to the row, over as many
// blocks as are resident; two kernels:
//   narrow    one or two rows of x: prepared by every block and kept in shared memory; the eight warps share the k axis, each
//             with a cp.async ring of its own that runs on across the block's row tiles, so that no warp waits for another
//             but once a tile, where the shares of k are joined.
//   streamed  more rows: x is prepared once by a kernel of its own, whose time the first loads of W hide, and comes through
//             the ring in runs of 256 k; kWr of the warps lie along the rows of W (x is read from L2 once for all of
//             them), 8 / kWr share the k axis.  float16 x against MX fp4 needs no preparation.
#include "ptx.cuh"
#include "internal.h"
#include "mx_format.cuh"
#include "prefix_attn.cuh"

namespace pto_b200 {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStepK = 256;              // k of one warp's step
constexpr int kStepBytes = kStepK / 2;   // bytes of a row of W in a step
constexpr int kPitch = kStepBytes + 16;  // 8 rows x 4 words of a quad's reads meet 32 distinct banks
constexpr int kNarrowPitch = kStepBytes;  // odd rows with their 64-byte halves exchanged: two rows x 4 lanes of a 16-byte read
constexpr int kXPitch = kStepK * 2 + 64; // two rows x 4 lanes of a 16-byte read phase likewise
constexpr int kStages = 3;               // of the streamed kernel's ring
constexpr int kNarrowStages = 3;         // of a warp's ring in the narrow kernel
constexpr int kNarrowSmem = 74 * 1024;   // of a block, for three an SM
constexpr int kNarrowMost = 112 * 1024;  // for two
constexpr int kSms = 148;

struct W4Args {
    const uint16_t *x;
    const uint8_t *w;
    const uint8_t *scale;
    const uint8_t *zero;
    void *y;
    int64_t x_stride;
    int m, n, k, group_shift, out_f32, out_bf16;
    int rows_each, rows_more; // rows of W a block owns; the first rows_more blocks one more
    const uint8_t *xp; // prepared x: runs of 256 k, x_run bytes each (streamed kernel)
    int x_run;
    int scale_async; // the scales of a step are 4, 8 or 16 aligned bytes a row: they ride in the ring
};

// bytes global -> shared, 4, 8 or 16, zeros where not live
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src, int size, bool live)
{
    const int n = live ? size : 0;
    if (size == 16) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    } else if (size == 8) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    } else {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    }
}

// eight e2m1 codes -> four float16 pairs (codes 2i, 2i + 1)
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&p)[4])
{
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
        : "r"(w));
}

// eight int4 codes as float16 subnormals: codes (0, 4) and (2, 6) times 2^-24, codes (1, 5) and (3, 7) times 2^-20
__device__ __forceinline__ void int4x8_to_f16(uint32_t w, uint32_t (&p)[4])
{
    p[0] = w & 0x000f000fu;
    p[1] = (w >> 8) & 0x000f000fu;
    p[2] = w & 0x00f000f0u;
    p[3] = (w >> 8) & 0x00f000f0u;
}

// Where a prepared run of 256 k of x lies: x_rows rows of kXPitch bytes, then per row 8 sums of x' (int4) and the factor
// 2^E (bfloat16), 36 bytes.  x_rows is m, and one row of zeros for the columns past it unless m fills the tiles.
constexpr int kXRow = kXPitch + 36;

// One warp prepares row `row`, k run `run` of x: eight elements a lane.
template <bool kBf16, bool kMx>
__device__ __forceinline__ void prepare_run(uint4 in, uint8_t *at, int x_rows, int row, int lane)
{
    uint32_t v[4] = {in.x, in.y, in.z, in.w};
    float *side = reinterpret_cast<float *>(at + x_rows * kXPitch) + row * 9;
    if constexpr (kBf16) {
        float2 f[4];
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[i] = unpack_16x2<true>(v[i]);
            top = fmaxf(top, fmaxf(fabsf(f[i].x), fabsf(f[i].y)));
        }
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top))); // not negative: ordered as integers
        // E = exponent of top - 14, kept where 2^E and 2^-E are normal numbers: -112 .. 113
        const int field = min(max(static_cast<int>(__float_as_uint(top) >> 23), 29), 254);
        const float inv = __uint_as_float(static_cast<uint32_t>(254 - (field - 14)) << 23);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = pack_16x2<false>(f[i].x * inv, f[i].y * inv);
        }
        if (lane == 0) {
            side[8] = __uint_as_float(static_cast<uint32_t>(field - 14) << 23);
        }
    }
    if constexpr (!kMx) { // sums of x' over runs of 32, for the zero points
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_16x2<false>(v[i]);
            sum += f.x + f.y;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if ((lane & 3) == 0) {
            side[lane >> 2] = sum;
        }
        // codes (i, i + 4) share a mask: k order (0, 4) (2, 6) (1, 5) (3, 7)
        const uint32_t y0 = v[0], y1 = v[1], y2 = v[2], y3 = v[3];
        v[0] = __byte_perm(y0, y2, 0x5410);
        v[1] = __byte_perm(y1, y3, 0x5410);
        v[2] = __byte_perm(y0, y2, 0x7632);
        v[3] = __byte_perm(y1, y3, 0x7632);
    }
    *reinterpret_cast<uint4 *>(at + row * kXPitch + lane * 16) = make_uint4(v[0], v[1], v[2], v[3]);
}

// where a lane finds its row of x in a prepared run, and the sums and factor of its columns of the result
template <int kMt>
struct LaneX {
    int row[kMt], col[kMt][2];
    __device__ __forceinline__ LaneX(int x_rows, int g, int t)
    {
#pragma unroll
        for (int c = 0; c < kMt; ++c) {
            row[c] = min(8 * c + g, x_rows - 1) * kXPitch + 16 * t;
            col[c][0] = x_rows * kXPitch + min(8 * c + 2 * t, x_rows - 1) * 36;
            col[c][1] = x_rows * kXPitch + min(8 * c + 2 * t + 1, x_rows - 1) * 36;
        }
    }
};

// 16 rows of W times the prepared run at `xs`: acc += .  `ws`: the lane's first word of the run's codes (row g, word t),
// `ss`, `zs`: the run's scales and zeros of row g (rows 16 bytes apart); blks: runs of 32 that exist.  A group of kG runs of
// 32 is summed before it is scaled.
template <bool kBf16, bool kMx, int kG, int kMt>
__device__ __forceinline__ void run_product(float (&acc)[kMt][4], const uint32_t *ws, const uint8_t *ss, const uint8_t *zs,
                                            const uint8_t *xs, const LaneX<kMt> &lx, bool zero, int blks)
{
    float f[kMt][2]; // 2^E of the lane's columns
#pragma unroll
    for (int c = 0; c < kMt; ++c) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f[c][j] = kBf16 ? *reinterpret_cast<const float *>(xs + lx.col[c][j] + 32) : 1.0f;
        }
    }
    auto group = [&](int first) {
        float d[kMt][4], e[kMt][4];
#pragma unroll
        for (int b = 0; b < kG; ++b) {
            const int blk = first + b;
            const uint32_t w0 = ws[blk * 4], w1 = ws[blk * 4 + 8 * kPitch / 4];
            uint32_t lo[4], hi[4];
            if constexpr (kMx) {
                e2m1x8_to_f16(w0, lo);
                e2m1x8_to_f16(w1, hi);
            } else {
                int4x8_to_f16(w0, lo);
                int4x8_to_f16(w1, hi);
            }
#pragma unroll
            for (int c = 0; c < kMt; ++c) {
                const uint4 xf = *reinterpret_cast<const uint4 *>(xs + lx.row[c] + blk * 64);
                if (b == 0) {
                    mma_16816_first<false>(d[c], lo[0], hi[0], lo[1], hi[1], xf.x, xf.y);
                } else {
                    mma_16816<false>(d[c], lo[0], hi[0], lo[1], hi[1], xf.x, xf.y);
                }
                if constexpr (kMx) {
                    mma_16816<false>(d[c], lo[2], hi[2], lo[3], hi[3], xf.z, xf.w);
                } else if (b == 0) {
                    mma_16816_first<false>(e[c], lo[2], hi[2], lo[3], hi[3], xf.z, xf.w);
                } else {
                    mma_16816<false>(e[c], lo[2], hi[2], lo[3], hi[3], xf.z, xf.w);
                }
            }
        }
        float s[2], z[2] = {8.0f, 8.0f};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (kMx) {
                s[i] = __uint_as_float(static_cast<uint32_t>(ss[i * 128 + first]) << 23);
                s[i] = fmaf(s[i], 0.0f, s[i]); // 255: infinity times 0 plus itself is NaN; 0 stands for 0, not 2^-127
            } else {
                const int at = i * 128 + first / kG * 2;
                s[i] = unpack_16x2<kBf16>(*reinterpret_cast<const uint16_t *>(ss + at)).x;
                if (zero) {
                    z[i] = unpack_16x2<kBf16>(*reinterpret_cast<const uint16_t *>(zs + at)).x;
                }
            }
        }
#pragma unroll
        for (int c = 0; c < kMt; ++c) {
            float u[2] = {0.0f, 0.0f};
            if constexpr (!kMx) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int b = 0; b < kG; ++b) {
                        u[j] += *reinterpret_cast<const float *>(xs + lx.col[c][j] + (first + b) * 4);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = d[c][i];
                if constexpr (!kMx) { // the codes went in times 2^-24 and 2^-20
                    v = fmaf(v, 16777216.0f, fmaf(e[c][i], 1048576.0f, -z[i >> 1] * u[i & 1]));
                }
                // 2^E before the scale: no product leaves fp32's range that x and W keep in it
                acc[c][i] = fmaf(kBf16 ? v * f[c][i & 1] : v, s[i >> 1], acc[c][i]);
            }
        }
    };
    if (blks >= kStepK / 32) {
#pragma unroll
        for (int blk = 0; blk < kStepK / 32; blk += kG) {
            group(blk);
        }
    } else {
#pragma unroll 1
        for (int blk = 0; blk < blks; blk += kG) {
            group(blk);
        }
    }
}

// The same for one or two rows of x.  Of the product's eight columns, columns 0 .. 3 take the four groups of 32 of half a
// run for the first row of x, columns 4 .. 7 for the second: lane t of a quad feeds group t (16 consecutive bytes of codes,
// one shared-memory read), and the x operand of column c is zero but in the k places of lane c mod 4.  So a column sums one
// group over eight products, and scales are applied once per 128 k where the wide form does so per 32: 17 instead of about
// 50 instructions per 32 k and 16 rows of W (8192 x 8192, one row: 17.1 us in the wide form).
// ws: row g, 16 bytes 16 t; odd: 64 in odd rows, whose halves are exchanged; acc: rows g and g + 8, the lane's two groups; xs: x of group t, or zeros; side: sums and 2^E of
// x row t / 2
template <bool kBf16, bool kMx>
__device__ __forceinline__ void run_product_narrow(float (&acc)[2], const uint8_t *ws, const uint8_t *ss, const uint8_t *zs,
                                                   const uint8_t *xs, const float *side, int group_shift, bool zero, int t, int odd)
{
    const float f = kBf16 ? side[8] : 1.0f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint4 a4 = *reinterpret_cast<const uint4 *>(ws + ((half * 64) ^ odd)), b4 = *reinterpret_cast<const uint4 *>(ws + ((half * 64) ^ odd) + 8 * kNarrowPitch);
        const uint32_t wa[4] = {a4.x, a4.y, a4.z, a4.w}, wb[4] = {b4.x, b4.y, b4.z, b4.w};
        float d[4], e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t lo[4], hi[4];
            if constexpr (kMx) {
                e2m1x8_to_f16(wa[j], lo);
                e2m1x8_to_f16(wb[j], hi);
            } else {
                int4x8_to_f16(wa[j], lo);
                int4x8_to_f16(wb[j], hi);
            }
            const uint4 xf = *reinterpret_cast<const uint4 *>(xs + half * 256 + j * 16);
            if (j == 0) {
                mma_16816_first<false>(d, lo[0], hi[0], lo[1], hi[1], xf.x, xf.y);
                mma_16816_first<false>(e, lo[2], hi[2], lo[3], hi[3], xf.z, xf.w);
            } else {
                mma_16816<false>(d, lo[0], hi[0], lo[1], hi[1], xf.x, xf.y);
                mma_16816<false>(e, lo[2], hi[2], lo[3], hi[3], xf.z, xf.w);
            }
        }
        // the lane's columns: groups 2 (t mod 2) and + 1 of this half
        const int blk = half * 4 + (t & 1) * 2;
        float s[2][2], z[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (kMx) {
                const uint32_t v = *reinterpret_cast<const uint16_t *>(ss + i * 128 + blk);
                s[i][0] = __uint_as_float((v & 0xffu) << 23);
                s[i][1] = __uint_as_float((v >> 8) << 23);
                s[i][0] = fmaf(s[i][0], 0.0f, s[i][0]); // 255: infinity times 0 plus itself is NaN; 0 stands for 0, not 2^-127
                s[i][1] = fmaf(s[i][1], 0.0f, s[i][1]);
            } else {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int at = i * 128 + ((blk + j) >> (group_shift - 5)) * 2;
                    s[i][j] = unpack_16x2<kBf16>(*reinterpret_cast<const uint16_t *>(ss + at)).x;
                    z[i][j] = zero ? unpack_16x2<kBf16>(*reinterpret_cast<const uint16_t *>(zs + at)).x : 8.0f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v;
            if constexpr (kMx) {
                v = d[i] + e[i];
            } else {
                v = fmaf(d[i], 16777216.0f, fmaf(e[i], 1048576.0f, -z[i >> 1][i & 1] * side[blk + (i & 1)]));
            }
            acc[i >> 1] = fmaf(kBf16 ? v * f : v, s[i >> 1][i & 1], acc[i >> 1]);
        }
    }
}

// row of zeros (with its sums and factor) of one run
__device__ __forceinline__ void clear_last_row(uint8_t *at, int x_rows, int thread, int threads)
{
    for (int i = thread; i < kXPitch / 16 + 9; i += threads) {
        if (i < kXPitch / 16) {
            *reinterpret_cast<uint4 *>(at + (x_rows - 1) * kXPitch + i * 16) = make_uint4(0, 0, 0, 0);
        } else {
            reinterpret_cast<float *>(at + x_rows * kXPitch)[(x_rows - 1) * 9 + i - kXPitch / 16] = 0.0f;
        }
    }
}

// the scales (or zeros) of one row in one step, to a 16-byte slot
__device__ __forceinline__ void load_scales(uint32_t dst, const uint8_t *row, int64_t first, int64_t row_bytes, int bytes, bool live, bool async)
{
    if (async) { // k a multiple of 256: a step's scales are whole and aligned
        live = live && first < row_bytes;
        cp_async(dst, live ? row + first : row, bytes, live);
    } else { // any k: byte by byte
        for (int i = 0; i < bytes; ++i) {
            const uint32_t v = live && first + i < row_bytes ? row[first + i] : 0u;
            asm volatile("st.shared.u8 [%0], %1;" ::"r"(dst + i), "r"(v) : "memory");
        }
    }
}

template <bool kBf16>
__device__ __forceinline__ void store_y(const W4Args &a, int64_t at, float v)
{
    if (a.out_f32) {
        static_cast<float *>(a.y)[at] = v;
    } else {
        static_cast<uint16_t *>(a.y)[at] = static_cast<uint16_t>(pack_16x2<kBf16>(v, 0.0f));
    }
}

// ------------------------------------------------------------------ one or two rows

template <bool kMx>
__host__ __device__ constexpr int narrow_stage_bytes()
{
    return 16 * kNarrowPitch + (kMx ? 1 : 2) * 256;
}

constexpr int kNarrowCols = 3; // floats of a row in a warp's share: two columns, and one so that rows meet other banks
constexpr int kNarrowShare = 16 * kNarrowCols;

// shared memory: the warps' rings, two buffers of shares of k, x (all runs), zeros
template <bool kMx>
int narrow_smem(int m, int k)
{
    return kWarps * kNarrowStages * narrow_stage_bytes<kMx>() + 2 * kWarps * kNarrowShare * 4 +
           (k + kStepK - 1) / kStepK * ((m * kXRow + 15) & ~15) + 512;
}

template <bool kBf16, bool kMx>
__global__ void __launch_bounds__(kThreads, 3) w4_narrow_kernel(const __grid_constant__ W4Args a)
{
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int kStage = narrow_stage_bytes<kMx>();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    uint8_t *ring = smem + warp * kNarrowStages * kStage;
    float *shares = reinterpret_cast<float *>(smem + kWarps * kNarrowStages * kStage);
    uint8_t *xs = smem + kWarps * kNarrowStages * kStage + 2 * kWarps * kNarrowShare * 4;
    const int x_run = (a.m * kXRow + 15) & ~15;
    const int block = static_cast<int>(blockIdx.x);
    const int row_begin = block * a.rows_each + min(block, a.rows_more), row_end = row_begin + a.rows_each + (block < a.rows_more ? 1 : 0);
    const int tiles = (row_end - row_begin + 15) / 16;
    const int64_t row_bytes = a.k / 2;
    const int64_t row_scale = static_cast<int64_t>(a.k >> a.group_shift) * (kMx ? 1 : 2);
    const int scale_bytes = kMx ? 8 : 512 >> a.group_shift;
    const int runs = (a.k + kStepK - 1) / kStepK;
    const int mine = (runs - warp + kWarps - 1) / kWarps; // this warp's runs of a tile: warp, warp + 8, ..

    // what is loaded next: run `ahead_run` of tile `ahead_tile`, at `src` for this lane (row lane / 8, 16 bytes lane % 8)
    int ahead_tile = mine > 0 ? 0 : tiles, ahead_run = warp;
    const int64_t four_rows = 4 * row_bytes;
    const uint8_t *src = a.w + (row_begin + (lane >> 3)) * row_bytes + warp * kStepBytes + (lane & 7) * 16;
    const bool zeros = lane >= 16, has_scale = !zeros || (!kMx && a.zero != nullptr);
    const uint8_t *scale_src = (zeros ? a.zero : a.scale) + (row_begin + (lane & 15)) * row_scale + warp * scale_bytes;
    const uint32_t dst = smem_u32(ring) + (lane >> 3) * kNarrowPitch + (((lane & 7) * 16) ^ ((lane & 8) * 8)), scale_dst = smem_u32(ring) + 16 * kNarrowPitch + lane * 16;
    auto load_next = [&](int stage) {
        if (ahead_tile < tiles) {
            const int rows = row_end - row_begin - ahead_tile * 16; // of this tile
            const uint32_t to = stage * kStage;
            if (rows >= 16 && (ahead_run + 1) * kStepK <= a.k) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    cp_async(dst + to + i * 4 * kNarrowPitch, src + i * four_rows, 16, true);
                }
            } else { // the end of the rows or of k (a multiple of 32: chunks are whole)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool live = i * 4 + (lane >> 3) < rows && ahead_run * kStepBytes + (lane & 7) * 16 < row_bytes;
                    cp_async(dst + to + i * 4 * kNarrowPitch, live ? src + i * four_rows : a.w, 16, live);
                }
            }
            if (has_scale) {
                if (a.scale_async) { // k a multiple of 256: a step's scales are whole and aligned
                    const bool live = (lane & 15) < rows;
                    cp_async(scale_dst + to, live ? scale_src : a.scale, scale_bytes, live);
                } else { // any k: byte by byte
                    for (int i = 0; i < scale_bytes; ++i) {
                        const uint32_t v = (lane & 15) < rows && ahead_run * scale_bytes + i < row_scale ? scale_src[i] : 0u;
                        asm volatile("st.shared.u8 [%0], %1;" ::"r"(scale_dst + to + i), "r"(v) : "memory");
                    }
                }
            }
            ahead_run += kWarps;
            src += kWarps * kStepBytes;
            scale_src += kWarps * scale_bytes;
            if (ahead_run >= runs) {
                ahead_run = warp;
                ++ahead_tile;
                src += 16 * row_bytes - static_cast<int64_t>(mine) * kWarps * kStepBytes;
                scale_src += 16 * row_scale - static_cast<int64_t>(mine) * kWarps * scale_bytes;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the lane feeds column g if that is group t of a row of x that exists
    uint8_t *nothing = xs + runs * x_run;
    const bool feeds = (g & 3) == t && (g >> 2) < a.m;
    const int x_at = (g >> 2) * kXPitch + t * 64, side_at = a.m * kXPitch + min(t >> 1, a.m - 1) * 36;
#pragma unroll
    for (int s = 0; s < kNarrowStages - 1; ++s) {
        load_next(s);
    }
    // x: a warp prepares one row of one run at a time
    for (int i = warp; i < runs * a.m; i += kWarps) {
        const int run = i / a.m, row = i - run * a.m;
        const int64_t k0 = static_cast<int64_t>(run) * kStepK + lane * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k0 < a.k) {
            v = __ldg(reinterpret_cast<const uint4 *>(a.x + row * a.x_stride + k0));
        }
        prepare_run<kBf16, kMx>(v, xs + run * x_run, a.m, row, lane);
    }
    if (threadIdx.x < 32) {
        reinterpret_cast<uint4 *>(nothing)[threadIdx.x] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();

    int stage = 0;
    for (int tile = 0; tile < tiles; ++tile) {
        float narrow[2] = {0.0f, 0.0f};
        for (int j = 0; j < mine; ++j) {
            load_next(stage == 0 ? kNarrowStages - 1 : stage - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(kNarrowStages - 1) : "memory");
            __syncwarp();
            const uint8_t *base = ring + stage * kStage;
            const int run = warp + j * kWarps;
            const uint8_t *ss = base + 16 * kNarrowPitch + g * 16, *x = xs + run * x_run;
            // codes, scales and x past the end of k are zeros: no run is short
            run_product_narrow<kBf16, kMx>(narrow, base + g * kNarrowPitch + 16 * t, ss, ss + 256, feeds ? x + x_at : nothing,
                                           reinterpret_cast<const float *>(x + side_at), a.group_shift, a.zero != nullptr, t, (g & 1) * 64);
            __syncwarp(); // every lane has read the stage before it is loaded again
            stage = stage + 1 == kNarrowStages ? 0 : stage + 1;
        }
        // the warps' shares of k joined in a fixed order; the buffers alternate, so one barrier a tile is enough
        float *share = shares + (tile & 1) * kWarps * kNarrowShare;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            narrow[i] += __shfl_xor_sync(0xffffffffu, narrow[i], 1); // groups 0, 1 and 2, 3
            if ((t & 1) == 0) {
                share[warp * kNarrowShare + (g + 8 * i) * kNarrowCols + (t >> 1)] = narrow[i];
            }
        }
        __syncthreads();
        const int n0 = row_begin + tile * 16;
        for (int i = threadIdx.x; i < a.m * 16; i += kThreads) {
            const int col = i >> 4, row = i & 15;
            if (n0 + row < row_end) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    v += share[w * kNarrowShare + row * kNarrowCols + col];
                }
                store_y<kBf16>(a, static_cast<int64_t>(col) * a.n + n0 + row, v);
            }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ------------------------------------------------------------------ more rows

// rows of a prepared run: m and one of zeros where the last column tile has columns left over
__host__ __device__ inline int streamed_x_rows(int m)
{
    return m <= 8 ? (m < 8 ? m + 1 : 8) : (m <= 16 ? (m < 16 ? m + 1 : 16) : (m <= 32 ? (m < 32 ? m + 1 : 32) : (m < 64 ? m + 1 : 64)));
}
__host__ __device__ inline int streamed_x_run(int m)
{
    return (streamed_x_rows(m) * kXRow + 15) & ~15;
}

// one warp prepares one row of one run, in the layout of the streamed kernel's shared memory
template <bool kBf16, bool kMx>
__global__ void __launch_bounds__(kThreads) w4_prepare_kernel(const __grid_constant__ W4Args a, uint8_t *xp)
{
    programmatic_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int x_rows = streamed_x_rows(a.m);
    const int unit = static_cast<int>(blockIdx.x) * kWarps + warp, run = unit / x_rows, row = unit - run * x_rows;
    if (run >= (a.k + kStepK - 1) / kStepK) {
        return;
    }
    uint8_t *at = xp + static_cast<int64_t>(run) * a.x_run;
    if (row >= a.m) {
        clear_last_row(at, x_rows, lane, 32);
        return;
    }
    const int64_t k0 = static_cast<int64_t>(run) * kStepK + lane * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k0 < a.k) {
        v = __ldg(reinterpret_cast<const uint4 *>(a.x + row * a.x_stride + k0));
    }
    prepare_run<kBf16, kMx>(v, at, x_rows, row, lane);
}

// shared memory of a stage: W [kWk][16 kWr rows][kPitch], scales and zeros [kWk][16 kWr rows][16], kWk runs of x; the shares
// of k are joined in the ring's place
template <bool kMx, int kWr, int kMt>
struct Layout {
    static constexpr int kWk = kWarps / kWr;
    static constexpr int kRows = 16 * kWr;
    static constexpr int kW = kWk * kRows * kPitch;
    static constexpr int kScale = kWk * kRows * 16;
    static constexpr int kX = kW + (kMx ? 1 : 2) * kScale;
    static constexpr int kSums = kWk * 8 * kMt * kRows * 4;
    static __host__ __device__ int stage_bytes(int m) { return kX + kWk * streamed_x_run(m); }
    static int smem_bytes(int m)
    {
        const int ring = kStages * stage_bytes(m);
        return ring > kSums ? ring : kSums;
    }
};

// kG: runs of 32 k in a group of the scales
template <bool kBf16, bool kMx, int kG, int kWr, int kMt>
__global__ void __launch_bounds__(kThreads, kMt <= 4 ? 2 : 1) w4_streamed_kernel(const __grid_constant__ W4Args a)
{
    using L = Layout<kMx, kWr, kMt>;
    constexpr int kWk = L::kWk;
    constexpr bool kRaw = !kBf16 && kMx; // x as it is
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int wr = warp % kWr, wk = warp / kWr;
    const int block = static_cast<int>(blockIdx.x);
    const int row_begin = block * a.rows_each + min(block, a.rows_more), row_end = row_begin + a.rows_each + (block < a.rows_more ? 1 : 0);
    const int64_t row_bytes = a.k / 2;
    const int64_t row_scale = static_cast<int64_t>(a.k / (32 * kG)) * (kMx ? 1 : 2);
    constexpr int kScaleBytes = kMx ? 8 : 16 / kG; // of a row in a step
    const int iters = (a.k + kStepK * kWk - 1) / (kStepK * kWk);
    const int x_rows = streamed_x_rows(a.m), x_run = streamed_x_run(a.m), stage_bytes = L::stage_bytes(a.m);
    const LaneX<kMt> lx(x_rows, g, t);
    if (kRaw && x_rows > a.m) { // the row of zeros stays where it is
        for (int i = warp; i < kStages * kWk; i += kWarps) {
            clear_last_row(smem + i / kWk * stage_bytes + L::kX + i % kWk * x_run, x_rows, lane, 32);
        }
    }
    bool waited = false;

    for (int n0 = row_begin; n0 < row_end; n0 += L::kRows) {
        // ---- this thread's pieces of a stage: 16-byte chunk threadIdx % 8 of rows row0 + 32 i of the (step, row) list
        constexpr int kPieces = L::kRows * kWk * 8 / kThreads; // 4
        const uint8_t *src[kPieces];
        uint32_t live = 0;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int r = i * (kThreads / 8) + (threadIdx.x >> 3), row = r % L::kRows, step = r / L::kRows;
            src[i] = a.w + (n0 + row < row_end ? (n0 + row) * row_bytes : 0) + step * kStepBytes + (threadIdx.x & 7) * 16;
            live |= n0 + row < row_end ? 1u << i : 0u;
        }
        const int sr = threadIdx.x & 127, s_row = sr % L::kRows, s_step = sr / L::kRows; // 128 runs of scales, then of zeros
        const bool zeros = threadIdx.x >= 128, has_scale = !zeros || (!kMx && a.zero != nullptr), s_live = n0 + s_row < row_end;
        const uint8_t *scale_src = (zeros ? a.zero : a.scale) + (s_live ? (n0 + s_row) * row_scale : 0);
        auto load_w = [&](int it) {
            const uint32_t base = smem_u32(smem) + (it % kStages) * stage_bytes;
            const bool whole = (it + 1) * kStepK * kWk <= a.k;
#pragma unroll
            for (int i = 0; i < kPieces; ++i) {
                const int r = i * (kThreads / 8) + (threadIdx.x >> 3), step = r / L::kRows;
                const int64_t off = static_cast<int64_t>(it) * kWk * kStepBytes;
                // k is a multiple of 32: chunks are whole
                const bool ok = (live >> i & 1u) && (whole || off + step * kStepBytes + (threadIdx.x & 7) * 16 < row_bytes);
                cp_async(base + r * kPitch + (threadIdx.x & 7) * 16, ok ? src[i] + off : a.w, 16, ok);
            }
            if (has_scale) {
                load_scales(base + L::kW + (zeros ? L::kScale : 0) + sr * 16, scale_src, (static_cast<int64_t>(it) * kWk + s_step) * kScaleBytes,
                            row_scale, kScaleBytes, s_live, a.scale_async);
            }
        };
        auto load_x = [&](int it) {
            const uint32_t base = smem_u32(smem) + (it % kStages) * stage_bytes + L::kX;
            if constexpr (kRaw) {
                for (int i = threadIdx.x; i < kWk * a.m * 32; i += kThreads) { // 32 chunks of a row's run
                    const int c = i & 31, unit = i >> 5, step = unit % kWk, row = unit / kWk;
                    const int64_t k0 = (static_cast<int64_t>(it) * kWk + step) * kStepK + c * 8;
                    cp_async(base + step * x_run + row * kXPitch + c * 16, a.x + (k0 < a.k ? row * a.x_stride + k0 : 0), 16, k0 < a.k);
                }
            } else { // kWk prepared runs, one after another
                const int chunks = kWk * x_run / 16, have = ((a.k + kStepK - 1) / kStepK - it * kWk) * (x_run / 16);
                const uint8_t *from = a.xp + static_cast<int64_t>(it) * kWk * x_run;
                for (int i = threadIdx.x; i < chunks && i < have; i += kThreads) {
                    cp_async(base + i * 16, from + i * 16, 16, true);
                }
            }
        };
        auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };

        float acc[kMt][4];
#pragma unroll
        for (int c = 0; c < kMt; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[c][i] = 0.0f;
            }
        }
#pragma unroll
        for (int s = 0; s < kStages - 1; ++s) { // W does not depend on the preparation of x
            if (s < iters) {
                load_w(s);
            }
        }
        if (!kRaw && !waited) {
            programmatic_wait();
            waited = true;
        }
#pragma unroll
        for (int s = 0; s < kStages - 1; ++s) {
            if (s < iters) {
                load_x(s);
            }
            commit();
        }
        for (int it = 0; it < iters; ++it) {
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
            __syncthreads(); // stage `it` is there, and everybody is done with the stage that the next loads overwrite
            if (it + kStages - 1 < iters) {
                load_w(it + kStages - 1);
                load_x(it + kStages - 1);
            }
            commit();
            const uint8_t *base = smem + (it % kStages) * stage_bytes;
            const int row = wk * L::kRows + wr * 16 + g;
            const int left = (a.k - (it * kWk + wk) * kStepK) / 32;
            if (left > 0 && n0 + wr * 16 < row_end) {
                run_product<kBf16, kMx, kG, kMt>(acc, reinterpret_cast<const uint32_t *>(base + row * kPitch) + t, base + L::kW + row * 16,
                                                 base + L::kW + L::kScale + row * 16, base + L::kX + wk * x_run, lx, a.zero != nullptr, left);
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        // the shares of k joined in a fixed order: [share][column of x][row of W]
        float *sums = reinterpret_cast<float *>(smem);
        constexpr int kM = 8 * kMt;
#pragma unroll
        for (int c = 0; c < kMt; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sums[(wk * kM + 8 * c + 2 * t + (i & 1)) * L::kRows + wr * 16 + g + 8 * (i >> 1)] = acc[c][i];
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.m * L::kRows; i += kThreads) {
            const int col = i / L::kRows, row = i % L::kRows;
            if (n0 + row < row_end) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < kWk; ++w) {
                    v += sums[(w * kM + col) * L::kRows + row];
                }
                store_y<kBf16>(a, static_cast<int64_t>(col) * a.n + n0 + row, v);
            }
        }
        __syncthreads(); // the sums are read before the ring is loaded again
        if (kRaw && x_rows > a.m && n0 + L::kRows < row_end) { // the sums lay over the rows of zeros
            for (int i = warp; i < kStages * kWk; i += kWarps) {
                clear_last_row(smem + i / kWk * stage_bytes + L::kX + i % kWk * x_run, x_rows, lane, 32);
            }
        }
    }
}

// ------------------------------------------------------------------ launches

template <bool kBf16, bool kMx>
int launch_narrow(W4Args a, cudaStream_t stream)
{
    const int smem = narrow_smem<kMx>(a.m, a.k), tiles = (a.n + 15) / 16;
    const int most = smem <= kNarrowSmem ? 3 * kSms : 2 * kSms, blocks = tiles < most ? tiles : most;
    a.rows_each = a.n / blocks;
    a.rows_more = a.n % blocks;
    // the attribute is raised once per kernel and device: to the most that is ever asked
    const int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(&w4_narrow_kernel<kBf16, kMx>), kNarrowMost);
    if (rc != kOk) {
        return rc;
    }
    w4_narrow_kernel<kBf16, kMx><<<blocks, kThreads, smem, stream>>>(a);
    return check_launch();
}

template <bool kBf16, bool kMx, int kG, int kWr, int kMt>
int launch_streamed(W4Args a, int blocks, uint8_t *workspace, cudaStream_t stream)
{
    using L = Layout<kMx, kWr, kMt>;
    const void *kernel = reinterpret_cast<const void *>(&w4_streamed_kernel<kBf16, kMx, kG, kWr, kMt>);
    int rc = ensure_dynamic_smem(kernel, L::smem_bytes(8 * kMt));
    constexpr bool kRaw = !kBf16 && kMx;
    if (!kRaw && rc == kOk) {
        a.xp = workspace;
        const int units = (a.k + kStepK - 1) / kStepK * streamed_x_rows(a.m);
        w4_prepare_kernel<kBf16, kMx><<<(units + kWarps - 1) / kWarps, kThreads, 0, stream>>>(a, workspace);
        rc = check_launch();
    }
    if (rc != kOk) {
        return rc;
    }
    a.rows_each = a.n / blocks;
    a.rows_more = a.n % blocks;
    return launch_overlapped(&w4_streamed_kernel<kBf16, kMx, kG, kWr, kMt>, static_cast<unsigned>(blocks), kThreads, L::smem_bytes(a.m), stream, !kRaw, a);
}

template <bool kBf16, bool kMx, int kG>
int launch_rows(W4Args a, uint8_t *workspace, cudaStream_t stream)
{
    // two blocks an SM, or one where that leaves a block fewer than 32 rows: every block reads all of x
    const int tiles = (a.n + 15) / 16;
    const int blocks = a.n >= 64 * kSms && a.m <= 32 ? 2 * kSms : (tiles < kSms ? tiles : kSms);
    const int rows = (a.n + blocks - 1) / blocks;
    a.x_run = streamed_x_run(a.m);
    if (a.m <= 8) {
        return rows <= 16   ? launch_streamed<kBf16, kMx, kG, 1, 1>(a, blocks, workspace, stream)
               : rows <= 32 ? launch_streamed<kBf16, kMx, kG, 2, 1>(a, blocks, workspace, stream)
               : rows <= 64 ? launch_streamed<kBf16, kMx, kG, 4, 1>(a, blocks, workspace, stream)
                            : launch_streamed<kBf16, kMx, kG, 8, 1>(a, blocks, workspace, stream);
    }
    if (a.m <= 16) {
        return rows <= 32   ? launch_streamed<kBf16, kMx, kG, 2, 2>(a, blocks, workspace, stream)
               : rows <= 64 ? launch_streamed<kBf16, kMx, kG, 4, 2>(a, blocks, workspace, stream)
                            : launch_streamed<kBf16, kMx, kG, 8, 2>(a, blocks, workspace, stream);
    }
    return a.m <= 32 ? launch_streamed<kBf16, kMx, kG, 8, 4>(a, blocks, workspace, stream)
                     : launch_streamed<kBf16, kMx, kG, 8, 8>(a, blocks, workspace, stream);
}

template <bool kBf16>
int launch_typed(const W4Args &a, bool mx, uint8_t *workspace, cudaStream_t stream)
{
    if (a.m <= 2 && (mx ? narrow_smem<true>(a.m, a.k) : narrow_smem<false>(a.m, a.k)) <= kNarrowMost) {
        return mx ? launch_narrow<kBf16, true>(a, stream) : launch_narrow<kBf16, false>(a, stream);
    }
    return mx                   ? launch_rows<kBf16, true, 1>(a, workspace, stream)
           : a.group_shift == 5 ? launch_rows<kBf16, false, 1>(a, workspace, stream)
           : a.group_shift == 6 ? launch_rows<kBf16, false, 2>(a, workspace, stream)
                                : launch_rows<kBf16, false, 4>(a, workspace, stream);
}

} // namespace

// room for the prepared x; not asked for where the call does without (few rows, or float16 x against MX fp4)
int64_t w4_matvec_workspace_bytes(int m, int k, bool mx)
{
    if (m <= 2 && (mx ? narrow_smem<true>(m, k) : narrow_smem<false>(m, k)) <= kNarrowMost) {
        return 0;
    }
    return static_cast<int64_t>((k + kStepK - 1) / kStepK) * streamed_x_run(m);
}

int launch_w4_matvec(const uint16_t *x, int64_t x_stride, const uint8_t *w, const void *scale, const uint16_t *zero, void *y,
                     int m, int n, int k, int group, bool bf16, bool mx, bool out_f32, void *workspace, int64_t workspace_bytes,
                     cudaStream_t stream)
{
    if (workspace_bytes < w4_matvec_workspace_bytes(m, k, mx) || (workspace == nullptr && w4_matvec_workspace_bytes(m, k, mx) > 0)) {
        set_error_text("w4_matvec: the workspace is smaller than pto_b200_w4_matvec_workspace_bytes says");
        return kErrBadArgument;
    }
    W4Args a = {};
    a.x = x;
    a.w = w;
    a.scale = static_cast<const uint8_t *>(scale);
    a.zero = reinterpret_cast<const uint8_t *>(zero);
    a.y = y;
    a.x_stride = x_stride;
    a.m = m;
    a.n = n;
    a.k = k;
    a.group_shift = group == 32 ? 5 : (group == 64 ? 6 : 7);
    a.out_f32 = out_f32;
    a.scale_async = k % kStepK == 0 && ((reinterpret_cast<uintptr_t>(scale) | reinterpret_cast<uintptr_t>(zero)) & 15u) == 0;
    return bf16 ? launch_typed<true>(a, mx, static_cast<uint8_t *>(workspace), stream)
                : launch_typed<false>(a, mx, static_cast<uint8_t *>(workspace), stream);
}

} // namespace pto_b200
