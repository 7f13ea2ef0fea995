// Products of a few 16-bit rows with a matrix of 4-bit weights: y[m, n] = sum_k x[m, k] W[n, k], m <= 64.
//
//   MX fp4   W = e2m1(code) 2^(byte - 127), one scale byte per 32 k: the weights of the MX fp4 GEMM, byte for byte
//   int4     W = s (code - z), code 0 .. 15, one 16-bit s (and z; 8 without) per group of 32, 64 or 128 k
// two codes a byte, the lower k in the low nibble.  The sum of a group is taken on the codes (exact in 16 bits, fp32
// accumulation on the tensor core) and scaled once:  y += s_group * (sum over the group of (code - z) x).
//
// Bound by HBM: n k / 2 bytes of weights are read once, everything else is small.  A block owns 16 * kRt rows of W and its
// eight warps share the k axis, each with a cp.async ring of its own (256 k = 128 bytes of every row a stage), so that no
// warp waits for another before the sums are joined.  Weights are the 16-row operand of mma.m16n8k16, the rows of x its
// eight columns.  The order of k inside a group of 32 is free as long as both operands agree: lane t of a quad takes
// k = 8t .. 8t + 7 (one 32-bit word of codes), paired (i, i + 4), so that one shift and one mask give a pair.
#include "ptx.cuh"
#include "internal.h"
#include "mx_format.cuh"

namespace pto_b200 {

namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kStepK = 256;               // k a warp takes at a time
constexpr int kStepBytes = kStepK / 2;    // bytes of a row of W in a stage
constexpr int kPitch = kStepBytes + 16;   // 8 rows x 4 words of a quad's reads meet 32 distinct banks
constexpr int kStages = 3;

struct W4Args {
    const uint16_t *x;
    const uint8_t *w;
    const void *scale;
    const uint16_t *zero;
    void *y;
    int64_t x_stride;
    int m, n, k, group_shift, out_f32;
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// the four pairs (code i, code i + 4) of a word of eight codes, as 16-bit values
template <bool kBf16, bool kMx>
__device__ __forceinline__ void codes_to_pairs(uint32_t w, uint32_t (&p)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kMx) {
            // sign to the top of each half, exponent and mantissa below it; the value is the code's times 2^-14 (float16:
            // exact even where subnormal, undone at the end) or 2^-126 (bfloat16: undone here, fp32 sums would underflow)
            const uint32_t top = i == 3 ? w : w << (4 * (3 - i));
            if constexpr (kBf16) {
                p[i] = mul_16x2<true>((top & 0x80008000u) | ((top >> 6) & 0x01c001c0u), 0x7e807e80u);
            } else {
                p[i] = (top & 0x80008000u) | ((top >> 3) & 0x0e000e00u);
            }
        } else if constexpr (kBf16) {
            // 0x4300 | code = 128 + code; minus 136 = code - 8, exact
            const uint32_t v = ((i == 0 ? w : w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
            asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(v), "r"(0x43084308u));
        } else {
            // 0x6400 | code = 1024 + code; minus 1032 = code - 8, exact
            const uint32_t v = ((i == 0 ? w : w >> (4 * i)) & 0x000f000fu) | 0x64006400u;
            asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(v), "r"(0x64086408u));
        }
    }
}

// kRt: tiles of 16 rows of W a block owns; kMt: tiles of 8 rows of x
template <bool kBf16, bool kMx, bool kZero, int kRt, int kMt>
__global__ void __launch_bounds__(kThreads) w4_matvec_kernel(const __grid_constant__ W4Args a)
{
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int kStageBytes = 16 * kRt * kPitch;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16 * kRt;
    const int64_t row_bytes = a.k / 2;
    const int groups = a.k >> a.group_shift;
    const int steps = (a.k + kStepK - 1) / kStepK;
    const uint32_t ring = smem_u32(smem) + warp * kStages * kStageBytes;

    auto load = [&](int step, int stage) {
        if (step < steps) {
            const uint32_t base = ring + stage * kStageBytes;
#pragma unroll
            for (int i = 0; i < 4 * kRt; ++i) { // 128 chunks of 16 bytes per 16 rows
                const int c = i * 32 + lane;
                const int r = c >> 3, at = (c & 7) * 16;
                const int64_t col = static_cast<int64_t>(step) * kStepBytes + at;
                const bool live = n0 + r < a.n && col < row_bytes; // k is a multiple of 32: chunks are whole
                cp_async16(base + r * kPitch + at, a.w + (live ? (n0 + r) * row_bytes + col : 0), live ? 16 : 0);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float acc[kRt][kMt][4];
#pragma unroll
    for (int r = 0; r < kRt; ++r) {
#pragma unroll
        for (int c = 0; c < kMt; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[r][c][i] = 0.0f;
            }
        }
    }
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
        load(warp + s * kWarps, s);
    }
    int stage = 0;
    for (int step = warp; step < steps; step += kWarps) {
        load(step + (kStages - 1) * kWarps, stage == 0 ? kStages - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        const uint32_t base = ring + stage * kStageBytes;
#pragma unroll 2
        for (int blk = 0; blk < kStepK / 32; ++blk) {
            const int k0 = step * kStepK + blk * 32;
            if (k0 >= a.k) {
                break;
            }
            // x: eight k of row 8c + g as pairs (i, i + 4)
            uint32_t xf[kMt][4];
#pragma unroll
            for (int c = 0; c < kMt; ++c) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (8 * c + g < a.m) {
                    v = *reinterpret_cast<const uint4 *>(a.x + (8 * c + g) * a.x_stride + k0 + 8 * t);
                }
                xf[c][0] = __byte_perm(v.x, v.z, 0x5410);
                xf[c][1] = __byte_perm(v.x, v.z, 0x7632);
                xf[c][2] = __byte_perm(v.y, v.w, 0x5410);
                xf[c][3] = __byte_perm(v.y, v.w, 0x7632);
            }
            // zero points other than 8: (code - z) x = (code - 8) x + (8 - z) x, the sum of x by a product with ones
            float xsum[kMt][2];
            if constexpr (kZero) {
                constexpr uint32_t kOnes = kBf16 ? 0x3f803f80u : 0x3c003c00u;
#pragma unroll
                for (int c = 0; c < kMt; ++c) {
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_16816<kBf16>(d, kOnes, kOnes, kOnes, kOnes, xf[c][0], xf[c][1]);
                    mma_16816<kBf16>(d, kOnes, kOnes, kOnes, kOnes, xf[c][2], xf[c][3]);
                    xsum[c][0] = d[0];
                    xsum[c][1] = d[1];
                }
            }
            const int grp = k0 >> a.group_shift;
#pragma unroll
            for (int r = 0; r < kRt; ++r) {
                uint32_t lo[4], hi[4];
                uint32_t w0, w1;
                const uint32_t at = base + (16 * r + g) * kPitch + blk * 16 + 4 * t;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w0) : "r"(at) : "memory");
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w1) : "r"(at + 8 * kPitch) : "memory");
                codes_to_pairs<kBf16, kMx>(w0, lo);
                codes_to_pairs<kBf16, kMx>(w1, hi);
                float s[2], z[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int row = min(n0 + 16 * r + g + 8 * i, a.n - 1);
                    const int64_t at_s = static_cast<int64_t>(row) * groups + grp;
                    if constexpr (kMx) {
                        s[i] = e8m0_value(static_cast<const uint8_t *>(a.scale)[at_s]);
                    } else {
                        s[i] = unpack_16x2<kBf16>(static_cast<const uint16_t *>(a.scale)[at_s]).x;
                    }
                    if constexpr (kZero) {
                        z[i] = 8.0f - unpack_16x2<kBf16>(a.zero[at_s]).x;
                    }
                }
#pragma unroll
                for (int c = 0; c < kMt; ++c) {
                    float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_16816<kBf16>(d, lo[0], hi[0], lo[1], hi[1], xf[c][0], xf[c][1]);
                    mma_16816<kBf16>(d, lo[2], hi[2], lo[3], hi[3], xf[c][2], xf[c][3]);
                    if constexpr (kZero) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            d[i] = fmaf(z[i >> 1], xsum[c][i & 1], d[i]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[r][c][i] = fmaf(d[i], s[i >> 1], acc[r][c][i]);
                    }
                }
            }
        }
        __syncwarp();
        stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // the warps' shares of k joined in a fixed order: [warp][column of x][row of W]
    float *sums = reinterpret_cast<float *>(smem);
    constexpr int kN = 16 * kRt, kM = 8 * kMt;
#pragma unroll
    for (int r = 0; r < kRt; ++r) {
#pragma unroll
        for (int c = 0; c < kMt; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sums[(warp * kM + 8 * c + 2 * t + (i & 1)) * kN + 16 * r + g + 8 * (i >> 1)] = acc[r][c][i];
            }
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kM * kN; i += kThreads) {
        const int col = i / kN, row = i % kN;
        if (col < a.m && n0 + row < a.n) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                v += sums[(w * kM + col) * kN + row];
            }
            if constexpr (kMx && !kBf16) {
                v *= 16384.0f; // the codes went in as 2^-14 times their values
            }
            const int64_t to = static_cast<int64_t>(col) * a.n + n0 + row;
            if (a.out_f32) {
                static_cast<float *>(a.y)[to] = v;
            } else {
                static_cast<uint16_t *>(a.y)[to] = static_cast<uint16_t>(pack_16x2<kBf16>(v, 0.0f));
            }
        }
    }
}

template <bool kBf16, bool kMx, bool kZero, int kRt, int kMt>
int launch_tiles(const W4Args &a, cudaStream_t stream)
{
    constexpr int kRing = kWarps * kStages * 16 * kRt * kPitch;
    constexpr int kSums = kWarps * 8 * kMt * 16 * kRt * 4;
    constexpr int kSmem = kRing > kSums ? kRing : kSums;
    const int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(&w4_matvec_kernel<kBf16, kMx, kZero, kRt, kMt>), kSmem);
    if (rc != kOk) {
        return rc;
    }
    const int blocks = (a.n + 16 * kRt - 1) / (16 * kRt);
    w4_matvec_kernel<kBf16, kMx, kZero, kRt, kMt><<<blocks, kThreads, kSmem, stream>>>(a);
    return check_launch();
}

template <bool kBf16, bool kMx, bool kZero>
int launch_typed(const W4Args &a, cudaStream_t stream)
{
    return a.m <= 8    ? launch_tiles<kBf16, kMx, kZero, 1, 1>(a, stream)
           : a.m <= 16 ? launch_tiles<kBf16, kMx, kZero, 1, 2>(a, stream)
           : a.m <= 32 ? launch_tiles<kBf16, kMx, kZero, 1, 4>(a, stream)
                       : launch_tiles<kBf16, kMx, kZero, 1, 8>(a, stream);
}

} // namespace

int launch_w4_matvec(const uint16_t *x, int64_t x_stride, const uint8_t *w, const void *scale, const uint16_t *zero, void *y,
                     int m, int n, int k, int group, bool bf16, bool mx, bool out_f32, cudaStream_t stream)
{
    W4Args a;
    a.x = x;
    a.w = w;
    a.scale = scale;
    a.zero = zero;
    a.y = y;
    a.x_stride = x_stride;
    a.m = m;
    a.n = n;
    a.k = k;
    a.group_shift = group == 32 ? 5 : (group == 64 ? 6 : 7);
    a.out_f32 = out_f32;
    if (mx) {
        return bf16 ? launch_typed<true, true, false>(a, stream) : launch_typed<false, true, false>(a, stream);
    }
    if (zero != nullptr) {
        return bf16 ? launch_typed<true, false, true>(a, stream) : launch_typed<false, false, true>(a, stream);
    }
    return bf16 ? launch_typed<true, false, false>(a, stream) : launch_typed<false, false, false>(a, stream);
}

} // namespace pto_b200
