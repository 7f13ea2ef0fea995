// Attention of few query tokens per sequence over a paged cache, for a batch whose sequences share a prefix.
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q.k_j - m)  over the prefix's keys and the sequence's own keys.
//
// The prefix's keys are read once for the whole batch: for each kv head the rows are all (sequence, query token, head of
// the group), so a key feeds batch * tokens * group rows of a product.  A sequence's own keys feed tokens * group rows.
// Both parts are cut along the keys into pieces that run side by side; each piece leaves (sum p v, sum p, m) in fp32
// for its rows and a second kernel joins them:  o = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i.
//
// piece kernel (16 rows a block): four warps, each walking every fourth group of 16 keys of the piece with a cp.async
// ring of its own, so no warp waits for another until the piece ends.  A lane's operands come from 16-byte reads:
//   S = Q K^T   the order of the head dimension inside a block of 32 is free as long as Q and K agree: lane t of a quad
//               takes elements 8t .. 8t+7 of the block, two k steps of four.  Codes are multiplied unscaled (exact in
//               16 bits) and the block's power of two is applied to the fp32 sums: S += 2^e (q_blk . code_blk).
//   O += P V    16-bit rows: V transposed on the way out of shared memory (ldmatrix).  Codes: a product's eight columns are
//               head-dimension elements W g + i (g the lane's group, W = d / 8), so a lane reads W consecutive elements of
//               its four keys and nothing is transposed; V's scale depends on the key and is applied to the pair.
// Over an MX cache the products are in float16 for either type of q: a code pair converts in one instruction (to bfloat16 in
// four, which made the kernel half as fast).  bfloat16 rows of q are divided by a power of two that brings their largest
// element into [2^14, 2^15); elements down to 2^-31 of it keep every bit.  V's scales are exact in float16 between 2^-15
// and 2^7 (e4m3; e2m1 2^-23 .. 2^13); 16 keys with one outside take bfloat16 products if q is bfloat16.  With float16 queries V
// is rounded to float16, by one product of pairs where that has the scale, by way of 32 bits elsewhere.
// Softmax statistics and all sums are fp32; P is rounded to the products' type.
//
// The piece kernel is bound by HBM where pieces are long and by its start and end (4-5 thousand cycles before the first
// step, 2.5 thousand after the last, 1850 for 64 keys) where they are short: 1024 pieces of 256 to 512 float16 keys of 128
// elements, 201 MB, take 42 us (4.8 TB/s), 256 of MX fp8, 26 MB, 13.4 us.
#include "ptx.cuh"
#include "prefix_attn.cuh"

#include <type_traits>

namespace pto_b200 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStep = 16; // keys a warp takes at a time
constexpr int kRows = kPieceRows; // query rows of a block
constexpr int kSms = 148; // planning constant: what the cut along the keys aims at

__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 bytes global -> shared; what lies past the first `bytes` is not read and arrives as zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit()
{
    asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a)
{
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a)
{
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a)
{
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

__host__ __device__ inline int ceil_div(int a, int b)
{
    return (a + b - 1) / b;
}

// keys of one piece of a sequence with `len` own keys: a multiple of 64, so that the four warps share it evenly
__device__ __forceinline__ int own_chunk(int len, int splits, int least)
{
    const int c = ((len + splits - 1) / splits + 63) & ~63;
    return c < least ? least : c;
}

// a sequence's number of own keys: never negative, never more than the table (or the caller's bound) covers
__device__ __forceinline__ int own_len(const AttnArgs &a, int b)
{
    const int n = a.lens[b];
    return n < 0 ? 0 : (n > a.own_max ? a.own_max : n);
}

// ---- shared-memory image of 16 rows of RB bytes: 16-byte chunks, exclusive-or swizzled within 128-byte lines so that
// the lanes of one access phase meet distinct banks.  K is read a key per quad (rows g), V a key per lane of a quad
// (rows 2t, 2t + 1).
template <int RB, int kFmt>
__device__ __forceinline__ uint32_t swz_k(int row, int byte)
{
    const int chunk = (row * RB + byte) >> 4;
    const int x = RB == 256 ? (row & 1) * 4
                  : RB == 128 ? (kFmt == kKvMxFp8 ? (2 * row) & 6 : (row & 1) * 4)
                  : RB == 64 ? (kFmt == kKvMxFp4 ? (row >> 1) & 3 : 2 * ((row >> 1) & 1))
                             : (row >> 2) & 1;
    return static_cast<uint32_t>(((chunk ^ x) << 4) | (byte & 15));
}
template <int RB, int kFmt>
__device__ __forceinline__ uint32_t swz_v(int row, int byte)
{
    const int chunk = (row * RB + byte) >> 4;
    const int t = (row >> 1) & 3;
    const int x = kFmt <= kKvBf16 ? row & 7 : RB == 128 ? row & 6 : RB == 64 ? 2 * t : 2 * ((row >> 2) & 1);
    return static_cast<uint32_t>(((chunk ^ x) << 4) | (byte & 15));
}

template <int kD, int kFmt>
struct Stage {
    static constexpr int kRowBytes = kv_row_bytes(kFmt, kD);
    static constexpr int kRowsBytes = kStep * kRowBytes;
    static constexpr int kScaleBytes = kFmt >= kKvMxFp8 ? kStep * kD / 32 : 0; // per K or V
    static constexpr int kBytes = 2 * kRowsBytes + 2 * kScaleBytes;
    static constexpr int kCount = kFmt <= kKvBf16 ? (kD == 128 ? 2 : 4) : (kFmt == kKvMxFp8 ? 4 : 6);
    static constexpr int kMergePitch = kD + 8; // floats: the rows of a store meet other banks
    static constexpr int kMergeBytes = kWarps * kRows * kMergePitch * 4 + kWarps * kRows * 8;
    static constexpr int kRing = kWarps * kCount * kBytes;
    static constexpr int kSmem = kRing > kMergeBytes ? kRing : kMergeBytes;
};

// Scaled V operand: a pair of values of two keys times the keys' powers of two.  In float16, by one product of pairs, where
// scale_ok() allows it
__device__ __forceinline__ uint32_t scale_pair(uint32_t b0, uint32_t b1)
{
    return pack_16x2<false>(__uint_as_float(b0 << 23), __uint_as_float(b1 << 23));
}
// The same by way of 32 bits: one rounding for every code (NaN among e4m3's) and scale byte
template <bool kBf16>
__device__ __forceinline__ uint32_t scaled_any(uint32_t h, float s0, float s1)
{
    const float2 f = unpack_16x2<false>(h);
    return pack_16x2<kBf16>(f.x * s0, f.y * s1);
}
// Whether one float16 product gives code times 2^(byte - 127): for bfloat16 queries every bit of it, for float16 queries its
// rounding to float16, which takes a power of two that float16 has, 2^-24 (byte 103) to 2^15 (byte 142).
template <bool kBf16, int kFmt>
__device__ __forceinline__ bool scale_ok(uint32_t byte)
{
    return !kBf16 ? byte - 103u <= 39u : kFmt == kKvMxFp8 ? byte - 112u <= 22u : byte - 104u <= 36u;
}

template <bool kBf16, int kD, int kFmt>
__global__ void __launch_bounds__(kThreads, 3) prefix_attn_piece_kernel(const __grid_constant__ AttnArgs a, DeviceStatus *status)
{
    using St = Stage<kD, kFmt>;
    constexpr bool kMx = kFmt >= kKvMxFp8;
    constexpr bool kOp = kBf16 && !kMx; // the products' type is bfloat16
    constexpr int RB = St::kRowBytes;
    constexpr int kBlk = kD / 32;
    constexpr int kTiles = kD / 8; // column tiles of O
    // Probabilities relative to 2^-15 of the running maximum where they become float16 beside V of float16's range: at most 2^15, they
    // keep every bit down to 2^-29 of the largest (2^-14 otherwise; a key that outweighs many others must not cost them).
    // Sums over V of bfloat16's range stay as they are, or they could leave fp32's.
    constexpr float kLift = kBf16 ? 0.0f : 15.0f, kDrop = kBf16 ? 1.0f : 0x1p-15f;
    extern __shared__ __align__(128) uint8_t smem[];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;

    programmatic_trigger();
    // ---- which piece
    // (32-bit arithmetic throughout: a 64-bit division costs more than a step's products)
    const int prefix_items = a.prefix_wide ? 0 : a.prefix_splits * a.kv_heads * a.prefix_tiles;
    const int row_span = a.tokens * a.group; // rows of one sequence and kv head
    const bool own = static_cast<int>(blockIdx.x) >= prefix_items;
    uint32_t item = blockIdx.x - (own ? prefix_items : 0);
    const uint32_t tiles = own ? a.own_tiles : a.prefix_tiles;
    int64_t slot = item + (own ? static_cast<int64_t>(a.prefix_pieces) * a.kv_heads * a.prefix_tiles : 0);
    const int tile = static_cast<int>(item % tiles);
    item /= tiles;
    const int h = static_cast<int>(item % static_cast<uint32_t>(a.kv_heads));
    item /= static_cast<uint32_t>(a.kv_heads);
    int b = 0, k_begin, k_end, rows, len = 0;
    const int32_t *pages;
    if (!own) {
        k_begin = static_cast<int>(item) * a.prefix_chunk;
        k_end = min(k_begin + a.prefix_chunk, a.prefix_len);
        rows = a.batch * row_span;
        pages = a.prefix_pages;
    } else {
        b = static_cast<int>(item % static_cast<uint32_t>(a.batch));
        const int split = static_cast<int>(item / static_cast<uint32_t>(a.batch));
        len = own_len(a, b);
        const int chunk = own_chunk(len, a.own_splits, a.own_min);
        k_begin = split * chunk;
        k_end = min(k_begin + chunk, len);
        rows = row_span;
        pages = a.table + b * a.table_stride;
        if (k_begin >= k_end) {
            programmatic_wait();
            return; // past this sequence's last piece: the joining kernel does not look here
        }
    }
    // the page of the step that is loaded next, read a step before
    const int steps = ceil_div(k_end - k_begin, kStep);
    int next_page = warp < steps ? pages[(k_begin + warp * kStep) >> a.page_shift] : 0;

    // ---- this lane's two rows: g and g + 8 of the tile
    int limit[2];
    const uint16_t *q_row[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = tile * kRows + g + 8 * i;
        const bool live = r < rows;
        const int bb = own ? b : (live ? r / row_span : 0);
        const int in = live ? (own ? r : r - bb * row_span) : 0;
        const int tok = a.tokens == 1 ? 0 : in / a.group;
        q_row[i] = live ? a.q + bb * a.q_batch + tok * a.q_token + static_cast<int64_t>(h * a.group + in - tok * a.group) * a.q_head : nullptr;
        // own keys: token `tok` of `tokens` sees all but the last tokens - 1 - tok
        limit[i] = !live ? 0 : (own ? min(k_end, len - (a.tokens - 1 - tok)) : k_end);
    }
    // Q operands: block kb, words {step 0: low pair, high pair, step 1: low pair, high pair}
    uint32_t qf[kBlk][2][4];
#pragma unroll
    for (int kb = 0; kb < kBlk; ++kb) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (q_row[i] != nullptr) {
                v = *reinterpret_cast<const uint4 *>(q_row[i] + 32 * kb + 8 * t);
            }
            qf[kb][i][0] = v.x;
            qf[kb][i][1] = v.y;
            qf[kb][i][2] = v.z;
            qf[kb][i][3] = v.w;
        }
    }
    float row_scale[2] = {a.scale_log2, a.scale_log2};
    if constexpr (kBf16 && kMx) { // rows of q to float16, see above; a quad holds a row
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t top = 0; // the largest magnitudes of both halves
#pragma unroll
            for (int kb = 0; kb < kBlk; ++kb) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t v = qf[kb][i][j] & 0x7fff7fffu;
                    asm("max.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(v));
                }
            }
            top = max(top & 0x7fffu, top >> 16);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int field = min(max(static_cast<int>(top >> 7), 29), 254);
            const float inv = __uint_as_float(static_cast<uint32_t>(254 - (field - 14)) << 23);
            row_scale[i] *= __uint_as_float(static_cast<uint32_t>(field - 14) << 23);
#pragma unroll
            for (int kb = 0; kb < kBlk; ++kb) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = unpack_16x2<true>(qf[kb][i][j]);
                    qf[kb][i][j] = pack_16x2<false>(f.x * inv, f.y * inv);
                }
            }
        }
    }

    // ---- this warp's steps and ring
    const uint32_t ring = smem_u32(smem) + warp * St::kCount * St::kBytes;
    uint32_t bad_pages = 0; // bit s: the step in ring stage s lies in a page that does not exist
    auto load = [&](int step, int stage) {
        if (step < steps) {
            const int key = k_begin + step * kStep;
            const int64_t page = next_page;
            if (step + kWarps < steps) {
                next_page = pages[(key + kWarps * kStep) >> a.page_shift];
            }
            const bool ok = page >= 0 && page < a.num_pages;
            bad_pages = (bad_pages & ~(1u << stage)) | (ok ? 0u : 1u << stage);
            if (!ok) {
                if (lane == 0 && atomicCAS(&status->code, 0, kErrBadArgument) == 0) {
                    status->block = blockIdx.x;
                    status->where = 11;
                    status->detail = static_cast<int>(page);
                }
            }
            const int64_t row = (((ok ? page : 0) * a.kv_heads + h) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
            const int live = ok ? min(kStep, k_end - key) : 0; // rows past the end arrive as zeros
            const uint32_t base = ring + stage * St::kBytes;
            constexpr int kChunks = St::kRowsBytes / 16;
#pragma unroll
            for (int c0 = 0; c0 < kChunks; c0 += 32) {
                const int c = c0 + lane;
                if (kChunks >= 32 || c < kChunks) {
                    const int r = (c * 16) / RB, byte = (c * 16) % RB;
                    const int64_t off = row * RB + c * 16;
                    cp_async16(base + swz_k<RB, kFmt>(r, byte), a.k + off, r < live ? 16 : 0);
                    cp_async16(base + St::kRowsBytes + swz_v<RB, kFmt>(r, byte), a.v + off, r < live ? 16 : 0);
                }
            }
            if constexpr (St::kScaleBytes > 0) {
                // the scales of 16 rows that start at a multiple of 16 are one run of kScaleBytes, 16-byte aligned
                constexpr int kSc = St::kScaleBytes / 16;
                if (lane < 2 * kSc) {
                    const int c = lane % kSc;
                    const uint8_t *src = (lane < kSc ? a.ks : a.vs) + row * (kD / 32) + c * 16;
                    // scales past the end arrive as 0, not as whatever the cache holds there: 0 * 2^128 would be NaN
                    cp_async16(base + 2 * St::kRowsBytes + lane * 16, src, max(0, min(16, live * (kD / 32) - c * 16)));
                }
            }
        }
        cp_async_commit();
    };

    float o[kTiles][4];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            o[i][j] = 0.0f;
        }
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

#pragma unroll
    for (int s = 0; s < St::kCount - 1; ++s) {
        load(warp + s * kWarps, s);
    }
    int stage = 0;
    for (int step = warp; step < steps; step += kWarps) {
        {
            const int ahead = stage == 0 ? St::kCount - 1 : stage - 1;
            load(step + (St::kCount - 1) * kWarps, ahead);
        }
        cp_async_wait<St::kCount - 1>();
        __syncwarp();
        const uint32_t base = ring + stage * St::kBytes;
        const int key0 = k_begin + step * kStep;
        const bool bad = (bad_pages >> stage) & 1u;

        // ---- S = Q K^T
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[n][j] = 0.0f;
            }
            float2 sc[2][kBlk / 2]; // scales of the lane's two columns (keys 8n + 2t, + 1), two blocks each; byte 255: NaN
            if constexpr (kFmt >= kKvMxFp8) {
                const uint32_t at = base + 2 * St::kRowsBytes + (8 * n + 2 * t) * kBlk;
                if constexpr (kBlk == 4) {
                    const uint2 v = lds64(at);
                    sc[0][0] = e8m0x2_to_f32(v.x);
                    sc[0][1] = e8m0x2_to_f32(v.x >> 16);
                    sc[1][0] = e8m0x2_to_f32(v.y);
                    sc[1][1] = e8m0x2_to_f32(v.y >> 16);
                } else {
                    const uint32_t v = lds32(at);
                    sc[0][0] = e8m0x2_to_f32(v);
                    sc[1][0] = e8m0x2_to_f32(v >> 16);
                }
            }
#pragma unroll
            for (int kb = 0; kb < kBlk; ++kb) {
                uint32_t w[4];
                if constexpr (kFmt <= kKvBf16) {
                    const uint4 v = lds128(base + swz_k<RB, kFmt>(8 * n + g, 64 * kb + 16 * t));
                    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                    mma_16816<kOp>(s[n], qf[kb][0][0], qf[kb][1][0], qf[kb][0][1], qf[kb][1][1], w[0], w[1]);
                    mma_16816<kOp>(s[n], qf[kb][0][2], qf[kb][1][2], qf[kb][0][3], qf[kb][1][3], w[2], w[3]);
                } else {
                    if constexpr (kFmt == kKvMxFp8) {
                        const uint2 v = lds64(base + swz_k<RB, kFmt>(8 * n + g, 32 * kb + 8 * t));
                        e4m3x4_to_f16(v.x, w[0], w[1]);
                        e4m3x4_to_f16(v.y, w[2], w[3]);
                    } else {
                        e2m1x8_to_f16(lds32(base + swz_k<RB, kFmt>(8 * n + g, 16 * kb + 4 * t)), w);
                    }
                    float p[4];
                    mma_16816_first<false>(p, qf[kb][0][0], qf[kb][1][0], qf[kb][0][1], qf[kb][1][1], w[0], w[1]);
                    mma_16816<false>(p, qf[kb][0][2], qf[kb][1][2], qf[kb][0][3], qf[kb][1][3], w[2], w[3]);
                    const float f0 = kb & 1 ? sc[0][kb / 2].y : sc[0][kb / 2].x;
                    const float f1 = kb & 1 ? sc[1][kb / 2].y : sc[1][kb / 2].x;
                    s[n][0] = fmaf(p[0], f0, s[n][0]);
                    s[n][1] = fmaf(p[1], f1, s[n][1]);
                    s[n][2] = fmaf(p[2], f0, s[n][2]);
                    s[n][3] = fmaf(p[3], f1, s[n][3]);
                }
            }
        }

        // ---- running maximum and sum, log2 units
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = key0 + 8 * n + 2 * t + (j & 1);
                const bool seen = key < limit[j >> 1] && !bad;
                s[n][j] = seen ? s[n][j] * row_scale[j >> 1] : -INFINITY;
                mx[j >> 1] = fmaxf(mx[j >> 1], s[n][j]);
            }
        }
        float ref[2], lifted[2], alpha[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            const float m_new = fmaxf(m[i], mx[i]);
            ref[i] = m_new == -INFINITY ? 0.0f : m_new; // a row that has seen no key yet
            lifted[i] = ref[i] - kLift;
            alpha[i] = ex2(m[i] - ref[i]);
            m[i] = m_new;
            l[i] *= alpha[i];
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
                o[i][0] *= alpha[0];
                o[i][1] *= alpha[0];
                o[i][2] *= alpha[1];
                o[i][3] *= alpha[1];
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[n][j] = ex2(s[n][j] - lifted[j >> 1]);
                l[j >> 1] += s[n][j];
            }
        }
        // ---- O += P V
        const uint32_t vbase = base + St::kRowsBytes;
        if constexpr (!kMx) {
            const uint32_t p0 = pack_16x2<kOp>(s[0][0], s[0][1]), p1 = pack_16x2<kOp>(s[0][2], s[0][3]);
            const uint32_t p2 = pack_16x2<kOp>(s[1][0], s[1][1]), p3 = pack_16x2<kOp>(s[1][2], s[1][3]);
#pragma unroll
            for (int i = 0; i < kTiles; i += 2) { // 16 keys x 16 elements, transposed; lane: key lane % 16, elements 8 (lane / 16)
                uint32_t v0, v1, v2, v3;
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                             : "=r"(v0), "=r"(v1), "=r"(v2), "=r"(v3)
                             : "r"(vbase + swz_v<RB, kFmt>(lane & 15, 16 * (i + (lane >> 4))))
                             : "memory");
                mma_16816<kOp>(o[i], p0, p1, p2, p3, v0, v1);
                mma_16816<kOp>(o[i + 1], p0, p1, p2, p3, v2, v3);
            }
        } else {
            // keys 2t, 2t + 1, 2t + 8, 2t + 9 of the step, elements W g .. W g + W - 1
            constexpr int kWords = kFmt == kKvMxFp8 ? kD / 32 : kD / 64; // 32-bit words of a lane's elements, per key
            uint32_t x[4][kWords], sb[4];
            const uint32_t sbase = base + 2 * St::kRowsBytes + St::kScaleBytes + (g * (kD / 8)) / 32;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = 2 * t + (i & 1) + (i >> 1) * 8;
                const uint32_t at = vbase + swz_v<RB, kFmt>(key, g * kWords * 4);
                sb[i] = lds8(sbase + key * kBlk);
                if constexpr (kWords == 4) {
                    const uint4 v = lds128(at);
                    x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
                } else if constexpr (kWords == 2) {
                    const uint2 v = lds64(at);
                    x[i][0] = v.x, x[i][1] = v.y;
                } else {
                    x[i][0] = lds32(at);
                }
            }
            // kAny: V of any scale, and the products in q's type; otherwise in float16
            auto product = [&](auto any) {
                constexpr bool kAny = decltype(any)::value, kWide = kAny && kBf16;
                const uint32_t p0 = pack_16x2<kWide>(s[0][0], s[0][1]), p1 = pack_16x2<kWide>(s[0][2], s[0][3]);
                const uint32_t p2 = pack_16x2<kWide>(s[1][0], s[1][1]), p3 = pack_16x2<kWide>(s[1][2], s[1][3]);
                const uint32_t pair01 = scale_pair(sb[0], sb[1]), pair23 = scale_pair(sb[2], sb[3]);
                const float2 f01 = e8m0x2_to_f32(sb[0] | (sb[1] << 8)), f23 = e8m0x2_to_f32(sb[2] | (sb[3] << 8));
                auto scaled01 = [&](uint32_t h) { return kAny ? scaled_any<kWide>(h, f01.x, f01.y) : mul_16x2<false>(h, pair01); };
                auto scaled23 = [&](uint32_t h) { return kAny ? scaled_any<kWide>(h, f23.x, f23.y) : mul_16x2<false>(h, pair23); };
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    if constexpr (kFmt == kKvMxFp8) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) { // bytes 2c and 2c + 1 of the word: {key 0, key 1} side by side
                            uint32_t lo[2], hi[2];
                            e4m3x4_to_f16(__byte_perm(x[0][w], x[1][w], c ? 0x7362 : 0x5140), lo[0], lo[1]);
                            e4m3x4_to_f16(__byte_perm(x[2][w], x[3][w], c ? 0x7362 : 0x5140), hi[0], hi[1]);
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                mma_16816<kWide>(o[4 * w + 2 * c + e], p0, p1, p2, p3, scaled01(lo[e]), scaled23(hi[e]));
                            }
                        }
                    } else {
                        // even nibbles of both keys in one byte, then odd ones
                        uint32_t even_lo[4], odd_lo[4], even_hi[4], odd_hi[4];
                        e2m1x8_to_f16((x[0][w] & 0x0f0f0f0fu) | ((x[1][w] << 4) & 0xf0f0f0f0u), even_lo);
                        e2m1x8_to_f16(((x[0][w] >> 4) & 0x0f0f0f0fu) | (x[1][w] & 0xf0f0f0f0u), odd_lo);
                        e2m1x8_to_f16((x[2][w] & 0x0f0f0f0fu) | ((x[3][w] << 4) & 0xf0f0f0f0u), even_hi);
                        e2m1x8_to_f16(((x[2][w] >> 4) & 0x0f0f0f0fu) | (x[3][w] & 0xf0f0f0f0u), odd_hi);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            mma_16816<kWide>(o[8 * w + 2 * i], p0, p1, p2, p3, scaled01(even_lo[i]), scaled23(even_hi[i]));
                            mma_16816<kWide>(o[8 * w + 2 * i + 1], p0, p1, p2, p3, scaled01(odd_lo[i]), scaled23(odd_hi[i]));
                        }
                    }
                }
            };
            auto ok = [&](int i) { return scale_ok<kBf16, kFmt>(sb[i]); };
            bool plain = __all_sync(0xffffffffu, ok(0) && ok(1) && ok(2) && ok(3));
            if (!plain) { // zeros have scale byte 0 (those of keys past the end too): as plain as any
                bool zeros = true;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t any = 0;
#pragma unroll
                    for (int w = 0; w < kWords; ++w) {
                        any |= x[i][w] & (kFmt == kKvMxFp8 ? 0x7f7f7f7fu : 0x77777777u);
                    }
                    zeros = zeros && (ok(i) || (sb[i] == 0u && any == 0u));
                }
                plain = __all_sync(0xffffffffu, zeros);
            }
            if (plain) {
                product(std::false_type{});
            } else {
                product(std::true_type{});
            }
        }
        __syncwarp(); // every lane has read the stage before it is loaded again
        stage = stage + 1 == St::kCount ? 0 : stage + 1;
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- the four warps' sums joined through shared memory
    float *mo = reinterpret_cast<float *>(smem);                                       // [warp][row][d]
    float2 *ml = reinterpret_cast<float2 *>(smem + kWarps * kRows * St::kMergePitch * sizeof(float)); // [warp][row]
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (t == 0) {
            ml[warp * kRows + g + 8 * i] = make_float2(m[i], l[i]);
        }
        if constexpr (!kMx) { // columns 2t and 2t + 1 of tile n: elements 8n + 2t, + 1
            float *dst = mo + (warp * kRows + g + 8 * i) * St::kMergePitch + 2 * t;
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                *reinterpret_cast<float2 *>(dst + 8 * n) = make_float2(o[n][2 * i], o[n][2 * i + 1]);
            }
        } else { // columns 2t and 2t + 1 of every tile: elements W (2t + c) .. + W - 1
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float4 *dst = reinterpret_cast<float4 *>(mo + (warp * kRows + g + 8 * i) * St::kMergePitch + kTiles * (2 * t + c));
#pragma unroll
                for (int n = 0; n < kTiles / 4; ++n) {
                    dst[n] = make_float4(o[4 * n][2 * i + c], o[4 * n + 1][2 * i + c], o[4 * n + 2][2 * i + c], o[4 * n + 3][2 * i + c]);
                }
            }
        }
    }
    __syncthreads();
    {
        // eight threads a row, four elements of every 32 each
        const int r = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * 4;
        float top = -INFINITY, w[kWarps], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            top = fmaxf(top, ml[i * kRows + r].x);
        }
        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
            const float2 v = ml[i * kRows + r];
            w[i] = ex2(v.x - ref) * kDrop;
            sum += v.y * w[i];
        }
        float *dst = a.part_o + (slot * kRows + r) * kD + c0;
#pragma unroll
        for (int c = 0; c < kD; c += 32) {
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                const float4 v = *reinterpret_cast<const float4 *>(mo + (i * kRows + r) * St::kMergePitch + c0 + c);
                acc.x = fmaf(v.x, w[i], acc.x);
                acc.y = fmaf(v.y, w[i], acc.y);
                acc.z = fmaf(v.z, w[i], acc.z);
                acc.w = fmaf(v.w, w[i], acc.w);
            }
            *reinterpret_cast<float4 *>(dst + c) = acc;
        }
        if (c0 == 0) {
            a.part_ml[slot * kRows + r] = make_float2(top, sum);
        }
    }
    programmatic_wait(); // this grid is not complete before the wide kernel's, which the joining kernel reads as well
}

// Joins a row's pieces in a fixed order: kShare warps a row, each every kShare-th piece, then their sums.  The pieces'
// statistics are read first, side by side; the loads of the sums depend on nothing and overlap.  Bound by latency and, with
// many rows, by what finding the pieces takes: four warps a row where a row has many pieces, one where it has few.  (Joined
// by the last block of a sequence's own pieces instead, one kernel fewer but fewer warps too, 24 sequences of 4 x 16 rows
// took 42 us for 33.)
template <bool kBf16, int kD, int kShare>
__global__ void __launch_bounds__(kThreads) prefix_attn_join_kernel(const __grid_constant__ AttnArgs a, DeviceStatus *status)
{
    constexpr int kPer = kD / 32, kAhead = 8;
    __shared__ float sums[kWarps], accs[kWarps][kD];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = kShare == 1 ? 0 : warp;
    const uint32_t idx = kShare == 1 ? blockIdx.x * kWarps + warp : blockIdx.x; // output row: (batch, token, head)
    if (kShare == 1 && idx >= static_cast<uint32_t>(a.batch) * a.tokens * a.heads) {
        programmatic_wait();
        return;
    }
    const uint32_t row = idx / static_cast<uint32_t>(a.heads);
    const uint32_t head = idx - row * a.heads;
    const uint32_t b = a.tokens == 1 ? row : row / static_cast<uint32_t>(a.tokens), tok = row - b * a.tokens;
    const int len = own_len(a, b);
    // a length out of range is reported here, where every sequence comes by whatever the lengths' bound is
    if (tok == 0 && head == 0 && part == 0 && lane == 0 && a.lens[b] != len && atomicCAS(&status->code, 0, kErrBadArgument) == 0) {
        status->block = blockIdx.x;
        status->where = 12;
        status->detail = a.lens[b];
    }
    const uint32_t h = head / static_cast<uint32_t>(a.group), in = tok * a.group + head - h * a.group;
    const uint32_t prow = b * a.tokens * a.group + in;
    const int own_pieces = len > 0 ? ceil_div(len, own_chunk(len, a.own_splits, a.own_min)) : 0;
    const int pieces = a.prefix_pieces + own_pieces;
    // where piece 0 of the prefix and (own piece 0) - prefix_pieces own pieces keep this row; rows between pieces
    const int64_t prefix_step = static_cast<int64_t>(a.kv_heads) * a.prefix_tiles * kRows;
    const int64_t own_step = static_cast<int64_t>(a.batch) * a.kv_heads * a.own_tiles * kRows;
    const int64_t prefix_row = static_cast<int64_t>(h) * a.prefix_tiles * kRows + prow;
    const int64_t own_row = a.prefix_pieces * (prefix_step - own_step) + (static_cast<int64_t>(b) * a.kv_heads + h) * a.own_tiles * kRows + in;
    auto row_of = [&](int i) { return i < a.prefix_pieces ? prefix_row + i * prefix_step : own_row + i * own_step; };
    programmatic_wait();
    float top = -INFINITY;
    for (int i = lane; i < pieces; i += 32) {
        top = fmaxf(top, a.part_ml[row_of(i)].x);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    float acc[kPer], sum = 0.0f;
#pragma unroll
    for (int c = 0; c < kPer; ++c) {
        acc[c] = 0.0f;
    }
    // eight of the warp's pieces at a time: statistics a piece a lane, the sums of all of them on their way at once
    for (int first = part; first < pieces; first += kShare * kAhead) {
        const int mine = first + (lane & (kAhead - 1)) * kShare;
        float w = 0.0f;
        bool used = false; // no key of the piece for this row: its sums may not even have been written
        if (mine < pieces) {
            const float2 v = a.part_ml[row_of(mine)];
            used = !(v.x == -INFINITY && v.y == 0.0f);
            w = ex2(v.x - ref);
            sum = used && lane < kAhead ? fmaf(v.y, w, sum) : sum;
        }
        float x[kAhead][kPer];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (first + u * kShare < pieces) {
                const float *src = a.part_o + row_of(first + u * kShare) * kD + lane * kPer;
                if constexpr (kPer == 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(src);
                    x[u][0] = v.x, x[u][1] = v.y, x[u][2] = v.z, x[u][3] = v.w;
                } else {
                    const float2 v = *reinterpret_cast<const float2 *>(src);
                    x[u][0] = v.x, x[u][1] = v.y;
                }
            }
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, used);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const float weight = __shfl_sync(0xffffffffu, w, u);
            if (mask >> u & 1u) {
#pragma unroll
                for (int c = 0; c < kPer; ++c) {
                    acc[c] = fmaf(x[u][c], weight, acc[c]);
                }
            }
        }
    }
#pragma unroll
    for (int s = kAhead / 2; s > 0; s >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, s);
    }
    if constexpr (kShare > 1) {
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
            accs[warp][lane * kPer + c] = acc[c];
        }
        if (lane == 0) {
            sums[warp] = sum;
        }
        __syncthreads();
        if (warp != 0) {
            return;
        }
        sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
#pragma unroll
        for (int c = 0; c < kPer; ++c) {
            const int at = lane * kPer + c;
            acc[c] = (accs[0][at] + accs[1][at]) + (accs[2][at] + accs[3][at]);
        }
    } else {
        sum = __shfl_sync(0xffffffffu, sum, 0);
    }
    const bool none = top == -INFINITY && sum == 0.0f; // no key at all: zeros
    const float inv = none ? 0.0f : 1.0f / sum;
    uint32_t *dst = reinterpret_cast<uint32_t *>(a.o + static_cast<int64_t>(idx) * kD + lane * kPer);
    if constexpr (kPer == 4) {
        *reinterpret_cast<uint2 *>(dst) = make_uint2(pack_16x2<kBf16>(acc[0] * inv, acc[1] * inv), pack_16x2<kBf16>(acc[2] * inv, acc[3] * inv));
    } else {
        *dst = pack_16x2<kBf16>(acc[0] * inv, acc[1] * inv);
    }
    if (a.lse != nullptr && lane == 0) {
        a.lse[idx] = none ? -INFINITY : (log2f(sum) + top) * 0.6931471805599453f;
    }
}

// How the keys are cut.  About three blocks of 16 rows fit an SM; a piece is at least 64 keys (16 for each warp).  A prefix of
// many rows and keys goes to the wide kernel, one block per SM, in one wave where it can.
struct Plan {
    int prefix_tiles, prefix_splits, prefix_pieces, prefix_chunk, prefix_wide;
    int own_tiles, own_splits, own_min;
    int64_t slots, own_slots;
};

// The piece kernel takes 0.065 ns a key, kv head and tile of 16 rows, the wide kernel as much as two such tiles for 128 rows, and
// 10 to 15 us more before and after.  A pass with pieces against one with the wide kernel, us, on both sides of the rule's border
// and far from it; 8 heads of 128 elements, MX fp8:
//   32 rows    12.4 / 19.5 at 4096 keys, 35.4 / 48.3 at 32768 (pieces at any length)
//   64 rows    10.8 / 13.9 at 1024, 24.0 / 26.2 at 8192 | 35.3 / 30.7 at 12288, 78.4 / 50.2 at 32768
//   128 rows   14.9 / 19.2 at 1024, 25.2 / 26.9 at 4096 | 37.3 / 29.5 at 6144, 150 / 55 at 32768
//   256 rows   21.5 / 28.2 at 1024, 28.2 / 32.3 at 2048 | 44.6 / 35.4 at 4096, 259 / 81 at 32768
//   512 rows   32.8 / 37.1 at 1024 | 46.5 / 40.0 at 2048, 261 / 83 at 16384
// float16: 64 rows 20.3 / 23.4 at 8192 | 31.2 / 26.4 at 12288; 128 rows 21.0 / 24.7 at 4096 | 34.1 / 26.7 at 6144.  64 elements: 64
// rows 16.4 / 19.7 at 8192 | 24.3 / 22.6 at 12288, 128 rows 17.8 / 19.5 at 4096 | 26.1 / 21.5 at 6144.  Other heads, 128 rows: one
// 24.1 / 40.3 at 32768, 32 of them 32.8 / 35.4 at 1024 | 46.7 / 39.8 at 2048; 2 heads, 768 rows 23.2 / 28.4 at 2048 | 37.0 / 31.3 at 4096.
bool wants_wide(int rows, int kv_heads, int prefix_len)
{
    const int64_t tiles = ceil_div(rows, kRows), more = tiles - 2 * static_cast<int64_t>(ceil_div(rows, 128));
    return more > 0 && more * kv_heads * prefix_len > 16384 * ((tiles < 8 ? tiles : 8) + 6);
}

// up to so many pieces of more rows than run at once with four warps each: a warp a row (4096 rows of 9 pieces: 8.3 us for
// 15.8; 8 rows of 9: 3.4 us with four warps, 4.0 with one)
constexpr int kFewPieces = 16, kManyRows = 1024;

Plan make_plan(int batch, int tokens, int heads, int kv_heads, int prefix_len, int own_max)
{
    Plan p = {};
    const int row_span = tokens * (heads / kv_heads);
    const int target = 3 * kSms;
    if (prefix_len > 0) {
        const int rows = batch * row_span;
        p.prefix_tiles = ceil_div(rows, kRows);
        p.prefix_wide = wants_wide(rows, kv_heads, prefix_len);
        if (p.prefix_wide) {
            const bool pair = rows > 128;
            const int64_t units = static_cast<int64_t>(ceil_div(rows, pair ? 256 : 128)) * kv_heads;
            const int tiles = ceil_div(prefix_len, 128);
            int splits = units >= kSms ? 1 : static_cast<int>(kSms / units);
            splits = splits > tiles ? tiles : splits;
            const int per = ceil_div(tiles, splits);
            p.prefix_chunk = per * 128;
            p.prefix_splits = ceil_div(tiles, per);
            p.prefix_pieces = pair ? p.prefix_splits : 2 * p.prefix_splits;
        } else {
            const int64_t units = static_cast<int64_t>(p.prefix_tiles) * kv_heads;
            int64_t splits = (target + units - 1) / units;
            const int most = ceil_div(prefix_len, 64);
            splits = splits > most ? most : splits;
            p.prefix_chunk = (ceil_div(prefix_len, static_cast<int>(splits)) + 63) & ~63;
            p.prefix_splits = ceil_div(prefix_len, p.prefix_chunk);
            p.prefix_pieces = p.prefix_splits;
        }
    }
    p.own_tiles = ceil_div(row_span, kRows);
    p.own_min = 64;
    if (own_max > 0) {
        // as many pieces as make the waves of blocks shortest: a piece costs its keys and about 384 more (queries, first
        // loads, joining its warps: 9000 cycles against 1850 for 64 keys); long sequences are cut anyway, for the sake of uneven lengths
        const int64_t units = static_cast<int64_t>(p.own_tiles) * kv_heads * batch;
        const int most = ceil_div(own_max, 64);
        int best = 1;
        int64_t best_cost = -1;
        for (int waves = 1; waves <= 4; ++waves) { // the most pieces that fit in so many waves
            int64_t splits = waves * static_cast<int64_t>(target) / units;
            splits = splits < 1 ? 1 : (splits > most ? most : splits);
            const int64_t cost = (units * splits + target - 1) / target * (ceil_div(own_max, static_cast<int>(splits)) + 384);
            if (best_cost < 0 || cost < best_cost) {
                best = static_cast<int>(splits);
                best_cost = cost;
            }
        }
        const int least = ceil_div(own_max, 2048);
        p.own_splits = best < least ? least : best;
        if (p.own_splits * units >= target) {
            p.own_min = 256;
        }
    }
    p.own_slots = static_cast<int64_t>(p.own_splits) * p.own_tiles * batch * kv_heads;
    p.slots = static_cast<int64_t>(p.prefix_pieces) * p.prefix_tiles * kv_heads + p.own_slots;
    return p;
}

template <bool kBf16, int kD, int kFmt>
int launch_pieces(const AttnArgs &a, int64_t blocks, DeviceStatus *status, cudaStream_t stream)
{
    constexpr int kSmem = Stage<kD, kFmt>::kSmem;
    const int rc = ensure_dynamic_smem(reinterpret_cast<const void *>(&prefix_attn_piece_kernel<kBf16, kD, kFmt>), kSmem);
    if (rc != kOk) {
        return rc;
    }
    return launch_overlapped(&prefix_attn_piece_kernel<kBf16, kD, kFmt>, static_cast<unsigned>(blocks), kThreads, kSmem, stream,
                             a.prefix_wide != 0, a, status);
}

template <bool kBf16, int kD>
int launch_typed(int fmt, const AttnArgs &a, int64_t own_slots, DeviceStatus *status, cudaStream_t stream)
{
    if (a.prefix_wide) {
        const int rc = launch_prefix_wide(a, fmt, kD, kBf16, status, stream);
        if (rc != kOk) {
            return rc;
        }
    }
    const int64_t blocks = own_slots + (a.prefix_wide ? 0 : static_cast<int64_t>(a.prefix_splits) * a.kv_heads * a.prefix_tiles);
    if (blocks > 0) {
        const int rc = fmt == kKvMxFp8   ? launch_pieces<kBf16, kD, kKvMxFp8>(a, blocks, status, stream)
                       : fmt == kKvMxFp4 ? launch_pieces<kBf16, kD, kKvMxFp4>(a, blocks, status, stream)
                                         : launch_pieces<kBf16, kD, kBf16 ? kKvBf16 : kKvF16>(a, blocks, status, stream);
        if (rc != kOk) {
            return rc;
        }
    }
    const int64_t rows = static_cast<int64_t>(a.batch) * a.tokens * a.heads;
    const bool after = blocks > 0 || a.prefix_wide != 0;
    if (a.prefix_pieces + a.own_splits <= kFewPieces && rows > kManyRows) {
        return launch_overlapped(&prefix_attn_join_kernel<kBf16, kD, 1>, static_cast<unsigned>((rows + kWarps - 1) / kWarps), kThreads, 0, stream, after, a, status);
    }
    return launch_overlapped(&prefix_attn_join_kernel<kBf16, kD, kWarps>, static_cast<unsigned>(rows), kThreads, 0, stream, after, a, status);
}

} // namespace

int64_t prefix_attn_workspace_bytes(int batch, int tokens, int heads, int kv_heads, int d, int prefix_len, int own_max)
{
    return make_plan(batch, tokens, heads, kv_heads, prefix_len, own_max).slots * kRows * (d * 4 + 8);
}

int launch_prefix_attn(const KvCacheView &cache, const uint16_t *q, bool bf16, const int64_t q_strides[3],
                       const int32_t *prefix_pages, int prefix_len, const int32_t *table, int64_t table_stride,
                       const int32_t *lens, int own_max, int batch, int tokens, int heads, float scale,
                       uint16_t *o, float *lse, void *workspace, int64_t workspace_bytes, cudaStream_t stream)
{
    const Plan p = make_plan(batch, tokens, heads, cache.kv_heads, prefix_len, own_max);
    if (workspace_bytes < p.slots * kRows * (cache.d * 4 + 8) || (p.slots > 0 && workspace == nullptr)) {
        set_error_text("prefix_attn: the workspace is smaller than pto_b200_prefix_attn_workspace_bytes says");
        return kErrBadArgument;
    }
    if (p.slots > 0x7fffffffLL) {
        set_error_text("prefix_attn: too many rows and pieces for one call");
        return kErrTooLarge;
    }
    DeviceStatus *status = device_status_ptr();
    if (status == nullptr) {
        return kErrCuda;
    }
    AttnArgs a;
    a.k = static_cast<const uint8_t *>(cache.k);
    a.v = static_cast<const uint8_t *>(cache.v);
    a.ks = cache.k_scale;
    a.vs = cache.v_scale;
    a.q = q;
    a.q_batch = q_strides[0];
    a.q_token = q_strides[1];
    a.q_head = q_strides[2];
    a.prefix_pages = prefix_pages;
    a.table = table;
    a.lens = lens;
    a.table_stride = table_stride;
    a.num_pages = cache.num_pages;
    a.part_o = static_cast<float *>(workspace);
    a.part_ml = reinterpret_cast<float2 *>(a.part_o + p.slots * kRows * cache.d);
    a.o = o;
    a.lse = lse;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.page_shift = cache.page_shift;
    a.batch = batch;
    a.tokens = tokens;
    a.heads = heads;
    a.kv_heads = cache.kv_heads;
    a.group = heads / cache.kv_heads;
    a.prefix_len = prefix_len;
    a.own_max = own_max;
    a.prefix_tiles = p.prefix_tiles;
    a.prefix_splits = p.prefix_splits;
    a.prefix_pieces = p.prefix_pieces;
    a.prefix_wide = p.prefix_wide;
    a.prefix_chunk = p.prefix_chunk;
    a.own_tiles = p.own_tiles;
    a.own_splits = p.own_splits;
    a.own_min = p.own_min;
    if (cache.d == 128) {
        return bf16 ? launch_typed<true, 128>(cache.fmt, a, p.own_slots, status, stream)
                    : launch_typed<false, 128>(cache.fmt, a, p.own_slots, status, stream);
    }
    return bf16 ? launch_typed<true, 64>(cache.fmt, a, p.own_slots, status, stream)
                : launch_typed<false, 64>(cache.fmt, a, p.own_slots, status, stream);
}

} // namespace pto_b200
