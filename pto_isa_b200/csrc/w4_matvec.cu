// Products of a few 16-bit rows with a matrix of 4-bit weights: y[m, n] = sum_k x[m, k] W[n, k], m <= 64.
//
//   MX fp4   W = e2m1(code) 2^(byte - 127), one scale byte per 32 k: the weights of the MX fp4 GEMM, byte for byte
//   int4     W = s (code - z), code 0 .. 15, one 16-bit s (and z; 8 without) per group of 32, 64 or 128 k
// two codes a byte, the lower k in the low nibble.  The sum of 32 k is taken on the codes, exactly representable in
// float16, by the tensor core with fp32 accumulation, and scaled afterwards:
//   y += 2^E s (sum (code) x' - z sum x'),   x = 2^E x'
// x' is x in float16.  float16 rows go in as they are (E = 0).  bfloat16 rows have float16's precision and more range,
// so each run of 256 gets the power of two that brings its largest element into [2^14, 2^15): every element down to
// 2^-31 of the largest keeps all its bits, below that the error is at most 2^-39 of the largest (2^-25 against 2^14), far under
// the rounding of the fp32 sum.  (A largest below 2^-98 does not get there: 2^E stays at 2^-112, and errors at 2^-137.)  Weights go through float16 because one conversion instruction turns two e2m1 codes into a
// float16 pair, and an int4 code is the float16 subnormal code * 2^-24 after one mask; to bfloat16 both take three to
// four half-rate integer operations a pair.
//
// n k / 2 bytes of weights are read once, everything else is small; in practice the instructions that a word of weights takes
// on its way to the tensor core bound it (8192 x 8192 MX fp4, one row: 14.3 us, 2.5 TB/s, and 12.2 with W in L2; 16384 x 4096
// int4 groups of 64 with zeros, 7 rows: 18.4 us; 32003 x 4096 MX fp4, 16 rows: 29.4 us).  Weights are the 16-row operand of
// mma.m16n8k16, the rows of x its eight columns; the order of k inside 32 is free as long as both operands agree: lane t
// of a quad takes k = 8t .. 8t + 7 (one word of codes).  The rows of W are dealt out evenly, to the row, over as many
// blocks as are resident; two kernels:
//   narrow    one or two rows of x: prepared by every block and kept in shared memory; the eight warps share the k axis, each
//             with a cp.async ring of its own that runs on across the block's row tiles, so that no warp waits for another
//             but once a tile, where the shares of k are joined.
//   streamed  more rows: x is prepared once by a kernel of its own, whose time the first loads of W hide, and comes through
//             the ring in runs of 256 k (prepared by every block again, 7 rows took 24.6 us for 20.0); kWr of the warps lie along the rows of W (x is read from L2 once for all of
//             them), 8 / kWr share the k axis.
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
constexpr int kNarrowPitch = kStepBytes;  // odd rows with their 64-byte halves exchanged: two rows x 4 lanes of a 16-byte read
constexpr int kXPitch = kStepK * 2 + 64; // two rows x 4 lanes of a 16-byte read phase likewise
constexpr int kBoxBytes = 16 * kStepBytes; // a warp's 16 rows of W in a step
constexpr int kNarrowStages = 3;         // of a warp's ring in the narrow kernel
constexpr int kNarrowSmem = 74 * 1024;   // of a block, for three an SM
constexpr int kNarrowMost = 112 * 1024;  // for two
constexpr int kStreamedSmem = 112 * 1024; // of a block, for two an SM
constexpr int kStreamedMost = 224 * 1024; // for one
constexpr int kSms = 148;

struct W4Args {
    const uint16_t *x;
    const uint8_t *w;
    const uint8_t *scale;
    const uint8_t *zero;
    void *y;
    int64_t x_stride;
    int m, n, k, group_shift, out_f32;
    int rows_each, rows_more; // rows of W a block owns; the first rows_more blocks one more
    const uint8_t *xp; // prepared x: runs of 256 k, x_run bytes each (streamed kernel)
    int x_run, stages, tile_rows; // tile_rows: rows of W that a block takes at once
    int scale_async; // the scales of a step are 4, 8 or 16 aligned bytes a row
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

// eight int4 codes as float16 subnormals: codes (0, 4) and (2, 6) times 2^-24, codes (1, 5) and (3, 7) times 2^-20
__device__ __forceinline__ void int4x8_to_f16(uint32_t w, uint32_t (&p)[4])
{
    p[0] = w & 0x000f000fu;
    p[1] = (w >> 8) & 0x000f000fu;
    p[2] = w & 0x00f000f0u;
    p[3] = (w >> 8) & 0x00f000f0u;
}

// Where a prepared run of 256 k of x lies: x_rows rows of kXPitch bytes, then per row up to 8 sums of x' (int4) and the factor
// 2^E (bfloat16), 36 bytes.  x_rows is m, and one row of zeros for the columns past it unless m fills the tiles.
constexpr int kXRow = kXPitch + 36;

// One warp prepares row `row`, k run `run` of x: eight elements a lane.
template <bool kBf16, bool kMx, int kG>
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
    if constexpr (!kMx) { // sums of x' over kG runs of 32, for the zero points
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack_16x2<false>(v[i]);
            sum += f.x + f.y;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if constexpr (kG >= 2) {
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        }
        if constexpr (kG >= 4) {
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        }
        if ((lane & (4 * kG - 1)) == 0) {
            side[lane / (4 * kG)] = sum;
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

// The scales or zeros of one row of W in one step
template <bool kMx, int kG>
struct StepScales {
    static constexpr int kBytes = kMx ? 8 : 16 / kG;
    static constexpr int kWords = kBytes / 4;
    uint32_t v[kWords];

    __device__ __forceinline__ void read(const uint8_t *at) // shared memory
    {
        if constexpr (kWords == 4) {
            const uint4 u = *reinterpret_cast<const uint4 *>(at);
            v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
        } else if constexpr (kWords == 2) {
            const uint2 u = *reinterpret_cast<const uint2 *>(at);
            v[0] = u.x, v[1] = u.y;
        } else {
            v[0] = *reinterpret_cast<const uint32_t *>(at);
        }
    }
    // to shared memory from a row that begins anywhere; zeros past its `left` bytes
    static __device__ __forceinline__ void gather(uint32_t dst, const uint8_t *src, int64_t left)
    {
#pragma unroll
        for (int w = 0; w < kWords; ++w) {
            uint32_t u = 0;
#pragma unroll
            for (int b = 0; b < 4; b += kMx ? 1 : 2) {
                if (4 * w + b < left) {
                    u |= kMx ? static_cast<uint32_t>(__ldg(src + 4 * w + b)) << (8 * b)
                             : static_cast<uint32_t>(__ldg(reinterpret_cast<const uint16_t *>(src + 4 * w + b))) << (8 * b);
                }
            }
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + 4 * w), "r"(u) : "memory");
        }
    }
    // of group `at` of the step
    template <bool kBf16>
    __device__ __forceinline__ float value(int at) const
    {
        if constexpr (kMx) {
            const float2 f = e8m0x2_to_f32(v[at >> 2] >> (at & 2) * 8);
            return at & 1 ? f.y : f.x;
        } else {
            const float2 f = unpack_16x2<kBf16>(v[at >> 1]);
            return at & 1 ? f.y : f.x;
        }
    }
};

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

__device__ __forceinline__ uint32_t ld_shared(uint32_t at)
{
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}

// 16 rows of W times the prepared run at `xs`: acc += .  `ws`: where the lane's words of the run's codes are, row g, word t
// of 16-byte chunk 0 ^ g (128-byte rows, chunks exchanged by the low bits of the row); `ss`: the step's scales of row g, zeros
// 16 rows behind.  A group of kG runs of 32 is summed
// before it is scaled.  What lies past the end of k is zero in W and x.
template <bool kBf16, bool kMx, int kG, int kMt>
__device__ __forceinline__ void run_product(float (&acc)[kMt][4], uint32_t ws, const uint8_t *ss, const uint8_t *xs, const LaneX<kMt> &lx, bool zero)
{
    using Scales = StepScales<kMx, kG>;
    Scales scales[2], zeros[2]; // rows g and g + 8
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        scales[i].read(ss + i * 8 * Scales::kBytes);
        if (!kMx && zero) {
            zeros[i].read(ss + (i * 8 + 16) * Scales::kBytes);
        }
    }
    float f[kMt][2]; // 2^E of the lane's columns
#pragma unroll
    for (int c = 0; c < kMt; ++c) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            f[c][j] = kBf16 ? *reinterpret_cast<const float *>(xs + lx.col[c][j] + 32) : 1.0f;
        }
    }
#pragma unroll
    for (int first = 0; first < kStepK / 32; first += kG) {
        float d[kMt][4], e[kMt][4];
#pragma unroll
        for (int b = 0; b < kG; ++b) {
            const int blk = first + b;
            const uint32_t w0 = ld_shared(ws ^ (blk * 16)), w1 = ld_shared((ws ^ (blk * 16)) + 8 * kStepBytes);
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
            s[i] = scales[i].template value<kBf16>(first / kG);
            if (!kMx && zero) {
                z[i] = zeros[i].template value<kBf16>(first / kG);
            }
        }
#pragma unroll
        for (int c = 0; c < kMt; ++c) {
            float u[2] = {0.0f, 0.0f};
            if constexpr (!kMx) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    u[j] = *reinterpret_cast<const float *>(xs + lx.col[c][j] + first / kG * 4);
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
    }
}

// The same for one or two rows of x.  Of the product's eight columns, columns 0 .. 3 take the four groups of 32 of half a
// run for the first row of x, columns 4 .. 7 for the second: lane t of a quad feeds group t (16 consecutive bytes of codes,
// one shared-memory read), and the x operand of column c is zero but in the k places of lane c mod 4.  So a column sums one
// group over eight products, and scales are applied once per 128 k where the wide form does so per 32 (8192 x 8192 MX fp4, one
// row: 14.3 us, 45 warp instructions of the whole kernel per 32 k and 16 rows of W; 17.1 us in the wide form).
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
                const float2 two = e8m0x2_to_f32(v);
                s[i][0] = two.x;
                s[i][1] = two.y;
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

// row of zeros (with its sums and factor) of one run, by one warp
__device__ __forceinline__ void clear_last_row(uint8_t *at, int x_rows, int lane)
{
    for (int i = lane; i < kXPitch / 16 + 9; i += 32) {
        if (i < kXPitch / 16) {
            *reinterpret_cast<uint4 *>(at + (x_rows - 1) * kXPitch + i * 16) = make_uint4(0, 0, 0, 0);
        } else {
            reinterpret_cast<float *>(at + x_rows * kXPitch)[(x_rows - 1) * 9 + i - kXPitch / 16] = 0.0f;
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
int64_t narrow_smem(int m, int k)
{
    return kWarps * kNarrowStages * narrow_stage_bytes<kMx>() + 2 * kWarps * kNarrowShare * 4 +
           (static_cast<int64_t>(k) + kStepK - 1) / kStepK * ((m * kXRow + 15) & ~15) + 512;
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
        prepare_run<kBf16, kMx, 1>(v, xs + run * x_run, a.m, row, lane);
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
template <bool kBf16, bool kMx, int kG>
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
        clear_last_row(at, x_rows, lane);
        return;
    }
    const int64_t k0 = static_cast<int64_t>(run) * kStepK + lane * 8;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (k0 < a.k) {
        v = __ldg(reinterpret_cast<const uint4 *>(a.x + row * a.x_stride + k0));
    }
    prepare_run<kBf16, kMx, kG>(v, at, x_rows, row, lane);
}

constexpr int kMostStages = 4;
constexpr int kScaleSlots = 4;

// shared memory: `stages` times kWk boxes of up to 16 kWr rows x 256 k of W, then `stages` times kWk runs of x,
// then kScaleSlots steps of scales and zeros a warp, then the shares of k on their way to be joined
template <int kWr, int kMt>
struct Layout {
    static constexpr int kWk = kWarps / kWr;
    static constexpr int kRows = 16 * kWr;
    static constexpr int kSums = kWk * 8 * kMt * kRows * 4;
    static __host__ __device__ int x_bytes(int m) { return kWk * streamed_x_run(m); }
    template <bool kMx, int kG>
    static __host__ __device__ constexpr int scale_bytes() // of a warp and step
    {
        return (kMx ? 16 : 32) * StepScales<kMx, kG>::kBytes;
    }
    template <bool kMx, int kG>
    static int smem_bytes(int m, int stages)
    {
        return stages * (kWarps * kBoxBytes + x_bytes(m)) + kWarps * kScaleSlots * scale_bytes<kMx, kG>() + kSums + 1024;
    }
};


struct StreamedCtl {
    uint64_t full[kMostStages];
    uint32_t done[kMostStages]; // warps that have read the stage
    int abort;
};

// untiled copy global -> shared, completion on an mbarrier; 16-byte aligned addresses and size
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// kG: runs of 32 k in a group of the scales.
// The warp that is the last to have read a stage loads it again: nobody waits for a stage to become free.
template <bool kBf16, bool kMx, int kG, int kWr, int kMt>
__global__ void __launch_bounds__(kThreads, kMt <= 4 ? 2 : 1)
    w4_streamed_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ W4Args a, DeviceStatus *status)
{
    using L = Layout<kWr, kMt>;
    using Scales = StepScales<kMx, kG>;
    constexpr int kWk = L::kWk;
    extern __shared__ uint8_t smem_raw[];
    __shared__ StreamedCtl ctl;
    uint8_t *smem = smem_raw + (-smem_u32(smem_raw) & 1023u);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int wr = warp % kWr, wk = warp / kWr;
    const int block = static_cast<int>(blockIdx.x);
    const int row_begin = block * a.rows_each + min(block, a.rows_more), row_end = row_begin + a.rows_each + (block < a.rows_more ? 1 : 0);
    const int runs = (a.k + kStepK - 1) / kStepK, iters = (runs + kWk - 1) / kWk;
    const int steps = (row_end - row_begin + a.tile_rows - 1) / a.tile_rows * iters;
    const int stages = a.stages;
    const int x_run = a.x_run, x_rows = streamed_x_rows(a.m);
    uint8_t *x_ring = smem + stages * kWarps * kBoxBytes;
    uint8_t *scale_slots = x_ring + stages * L::x_bytes(a.m);
    float *sums = reinterpret_cast<float *>(scale_slots + kWarps * kScaleSlots * L::template scale_bytes<kMx, kG>());
    const LaneX<kMt> lx(x_rows, g, t);

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(&ctl.full[s], 1);
            ctl.done[s] = 0;
        }
        ctl.abort = 0;
        fence_mbar_init();
    }
    __syncthreads();

    // a warp announces a step, and loads W: a box of the block's rows for each of its runs of 256
    auto load_w = [&](int slot, int n0, int it) {
        const int have = min(kWk, runs - it * kWk);
        if (lane == 0) {
            mbar_arrive_expect_tx(&ctl.full[slot], static_cast<uint32_t>(have) * (a.tile_rows * kStepBytes + x_run));
        }
        __syncwarp();
        if (lane < have) {
            tma_load_2d(smem + slot * kWarps * kBoxBytes + lane * L::kRows * kStepBytes, &tmap_w, &ctl.full[slot], (it * kWk + lane) * kStepBytes, n0);
        }
    };
    auto load_x = [&](int slot, int it) { // runs lie one after another
        if (lane == 0) {
            bulk_load(smem_u32(x_ring) + slot * kWk * x_run, a.xp + static_cast<int64_t>(it) * kWk * x_run,
                      static_cast<uint32_t>(min(kWk, runs - it * kWk) * x_run), &ctl.full[slot]);
        }
    };
    // W does not depend on the preparation of x; x, prepared by the kernel before, is waited for
    int ahead_n0 = row_begin, ahead_it = 0; // of the step that is `stages` ahead
    if (warp == 0) {
        int n0 = row_begin, it = 0;
        for (int s = 0; s < stages && s < steps; ++s) {
            load_w(s, n0, it);
            it = it + 1 == iters ? 0 : it + 1;
            n0 += it == 0 ? a.tile_rows : 0;
        }
    }
    // The warp's own scales, 16 rows a step, and zeros run kScaleSlots - 1 steps ahead: lane 0 .. 15 a row's scales, 16 .. 31
    // its zeros, at `scale_src` for the step that comes next
    const bool zero = !kMx && a.zero != nullptr;
    const int64_t row_scale = static_cast<int64_t>(a.k / (32 * kG)) * (kMx ? 1 : 2);
    uint8_t *slots = scale_slots + warp * kScaleSlots * L::template scale_bytes<kMx, kG>();
    const uint32_t scale_dst = smem_u32(slots) + lane * Scales::kBytes;
    int scale_n0 = row_begin + 16 * wr + (lane & 15), scale_run = wk, scale_slot = 0;
    const uint8_t *scale_src = nullptr;
    auto scale_row = [&] { // rows past the end: any row, its result is not stored
        scale_src = (lane < 16 ? a.scale : a.zero) + min(scale_n0, a.n - 1) * row_scale + wk * Scales::kBytes;
    };
    scale_row();
    auto load_scales = [&] {
        if ((lane < 16 || zero) && scale_run < runs) {
            const uint32_t dst = scale_dst + scale_slot * L::template scale_bytes<kMx, kG>();
            if (a.scale_async) {
                cp_async(dst, scale_src, Scales::kBytes, true);
            } else {
                Scales::gather(dst, scale_src, row_scale - static_cast<int64_t>(scale_run) * Scales::kBytes);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        scale_slot = (scale_slot + 1) & (kScaleSlots - 1);
        scale_run += kWk;
        scale_src += kWk * Scales::kBytes;
        if (scale_run >= iters * kWk) {
            scale_run = wk;
            scale_n0 += a.tile_rows;
            scale_row();
        }
    };
    for (int i = 0; i < kScaleSlots - 1; ++i) {
        load_scales();
    }
    programmatic_wait();
    if (warp == 0) {
        int it = 0;
        for (int s = 0; s < stages && s < steps; ++s) {
            load_x(s, it);
            it = it + 1 == iters ? 0 : it + 1;
        }
    }
    for (int s = 0; s < stages; ++s) {
        ahead_it = ahead_it + 1 == iters ? 0 : ahead_it + 1;
        ahead_n0 += ahead_it == 0 ? a.tile_rows : 0;
    }

    int slot = 0, read_slot = 0, left = steps;
    uint32_t parity = 0;
    bool ok = true;
    const uint32_t lane_w = smem_u32(smem) + warp * kBoxBytes + g * (kStepBytes + 16) + 4 * t; // row g, chunk 0 ^ g
    for (int n0 = row_begin; n0 < row_end; n0 += a.tile_rows) {
        const int rows = min(a.tile_rows, row_end - n0);
        float acc[kMt][4];
#pragma unroll
        for (int c = 0; c < kMt; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[c][i] = 0.0f;
            }
        }
        for (int it = 0; it < iters; ++it) {
            load_scales();
            asm volatile("cp.async.wait_group %0;" ::"n"(kScaleSlots - 1) : "memory");
            if (ok) {
                ok = __all_sync(0xffffffffu, mbar_wait(&ctl.full[slot], parity, &ctl.abort));
            }
            __syncwarp(); // the scales of all lanes
            if (ok) {
                if (it * kWk + wk < runs && wr * 16 < rows) {
                    run_product<kBf16, kMx, kG, kMt>(acc, lane_w + slot * kWarps * kBoxBytes,
                                                     slots + read_slot * L::template scale_bytes<kMx, kG>() + g * Scales::kBytes, x_ring + (slot * kWk + wk) * x_run, lx, zero);
                }
                __syncwarp();
                uint32_t before = 0;
                if (lane == 0 && left > stages) {
                    asm volatile("atom.acq_rel.cta.shared::cta.add.u32 %0, [%1], 1;" : "=r"(before) : "r"(smem_u32(&ctl.done[slot])) : "memory");
                    if (before == kWarps - 1) {
                        ctl.done[slot] = 0;
                    }
                }
                if (__shfl_sync(0xffffffffu, before, 0) == kWarps - 1) { // everybody has read the stage
                    load_w(slot, ahead_n0, ahead_it);
                    load_x(slot, ahead_it);
                }
            }
            read_slot = (read_slot + 1) & (kScaleSlots - 1);
            --left;
            ahead_it = ahead_it + 1 == iters ? 0 : ahead_it + 1;
            ahead_n0 += ahead_it == 0 ? a.tile_rows : 0;
            slot = slot + 1 == stages ? 0 : slot + 1;
            parity ^= slot == 0 ? 1u : 0u;
        }
        // the shares of k joined in a fixed order: [share][column of x][row of W]
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
            if (row < rows) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < kWk; ++w) {
                    v += sums[(w * kM + col) * L::kRows + row];
                }
                store_y<kBf16>(a, static_cast<int64_t>(col) * a.n + n0 + row, v);
            }
        }
        if (n0 + a.tile_rows < row_end) {
            __syncthreads(); // the sums are read before they are written again
        }
    }
    if (__syncthreads_or(!ok)) { // a copy that never came
        for (int i = 0; i < 1024; ++i) {
            __nanosleep(1000); // copies in flight end before the shared memory is given back
        }
        if (threadIdx.x == 0 && atomicCAS(&status->code, 0, kErrDeviceWaitTimeout) == 0) {
            status->block = block;
            status->where = 6;
        }
        __syncthreads();
    }
}

// ------------------------------------------------------------------ launches

template <bool kBf16, bool kMx>
int launch_narrow(W4Args a, cudaStream_t stream)
{
    const int smem = static_cast<int>(narrow_smem<kMx>(a.m, a.k)), tiles = (a.n + 15) / 16;
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
    using L = Layout<kWr, kMt>;
    auto kernel = &w4_streamed_kernel<kBf16, kMx, kG, kWr, kMt>;
    int stages = kMostStages; // what two blocks an SM leave room for, or one
    const int room = L::template smem_bytes<kMx, kG>(a.m, 2) <= kStreamedSmem ? kStreamedSmem : kStreamedMost;
    while (stages > 2 && L::template smem_bytes<kMx, kG>(a.m, stages) > room) {
        --stages;
    }
    a.stages = stages;
    a.rows_each = a.n / blocks;
    a.rows_more = a.n % blocks;
    const int rows = a.rows_each + (a.rows_more > 0 ? 1 : 0), tiles = (rows + L::kRows - 1) / L::kRows;
    a.tile_rows = (rows + tiles - 1) / tiles;
    CUtensorMap tmap_w;
    DeviceStatus *status = device_status_ptr();
    if (status == nullptr) {
        return kErrCuda;
    }
    int rc = make_tmap_2d(&tmap_w, a.w, 1, static_cast<uint64_t>(a.n), static_cast<uint64_t>(a.k) / 2, static_cast<uint64_t>(a.k) / 2, static_cast<uint32_t>(a.tile_rows), kStepBytes, true);
    if (rc == kOk) {
        rc = ensure_dynamic_smem(reinterpret_cast<const void *>(kernel), kStreamedMost);
    }
    if (rc == kOk) {
        a.xp = workspace;
        const int units = (a.k + kStepK - 1) / kStepK * streamed_x_rows(a.m);
        w4_prepare_kernel<kBf16, kMx, kG><<<(units + kWarps - 1) / kWarps, kThreads, 0, stream>>>(a, workspace);
        rc = check_launch();
    }
    if (rc != kOk) {
        return rc;
    }
    return launch_overlapped(kernel, static_cast<unsigned>(blocks), kThreads, L::template smem_bytes<kMx, kG>(a.m, stages), stream, true, tmap_w, a, status);
}

template <bool kBf16, bool kMx, int kG>
int launch_rows(W4Args a, uint8_t *workspace, cudaStream_t stream)
{
    // two blocks an SM, or one where that leaves a block no more than 32 rows (every block reads all of x) or more rows of x
    // than two blocks' registers hold; three blocks of 80 registers: 24.6 us for 20.0 at 7 rows, 33.1 for 30.7 at 16
    const int tiles = (a.n + 15) / 16;
    const int blocks = a.n > 64 * kSms && a.m <= 32 ? 2 * kSms : (tiles < kSms ? tiles : kSms);
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

// room for the prepared x; none where every block prepares it for itself
int64_t w4_matvec_workspace_bytes(int m, int k, bool mx)
{
    if (m <= 2 && (mx ? narrow_smem<true>(m, k) : narrow_smem<false>(m, k)) <= kNarrowMost) {
        return 0;
    }
    return (static_cast<int64_t>(k) + kStepK - 1) / kStepK * streamed_x_run(m);
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
