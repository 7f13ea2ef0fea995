// The paged key / value cache: rows are quantised as they are written and read back as 16-bit tensors.
//
// A cache holds K and V as (pages, kv_heads, page_size, row) with a row of head_dim elements in 16 bits, in MX fp8
// (float8_e4m3fn) or MX fp4 (float4_e2m1, the lower index in the low nibble), the MX formats with one e8m0 scale byte per
// 32 elements in (pages, kv_heads, page_size, head_dim / 32).  For a block x of 32 elements
//     a = max |x|,  e = the smallest integer with a <= M 2^e (M = 448 or 6),  code = RNE(x 2^-e),  value = code 2^e:
// everything but the one rounding is exact, so a row's codes do not depend on who computes them.  A block that holds a
// NaN or an infinity gets the scale byte 255 and reads back as NaN throughout (e2m1 has no NaN of its own).
//
// Both kernels move bytes and are bound by HBM, the fp4 read about as much by its instructions.  Writing, a thread owns 16
// elements: 32 bytes of the source, half a scale block whose partner is one lane away.  Reading, it owns 8, so that every
// store instruction of a warp fills whole lines (16 elements a thread, the stores 32 bytes apart, took 40 us where this takes
// 32), in four rows of K and V at once (one row at a time: 36 us).  8 heads x 8 sequences x 4096 keys of 128 elements in MX
// fp8: 185 MB in 32 us, 5.7 TB/s; 512 new keys each: 26 MB in 7.3 us.
#include "ptx.cuh"
#include "internal.h"
#include "mx_format.cuh"

namespace pto_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;     // elements a thread of the write kernel owns
constexpr int kReadRows = 4; // rows of K and of V a thread of the read kernel has on their way

__device__ __forceinline__ void report_index(DeviceStatus *status, int where, int detail)
{
    if (atomicCAS(&status->code, 0, kErrBadArgument) == 0) {
        status->block = blockIdx.x;
        status->where = where;
        status->detail = detail;
    }
}

// quantises 16 elements (8 words of two); both lanes of a block's pair call it
template <bool kBf16, int kFmt>
__device__ __forceinline__ void encode16(const uint32_t (&w)[8], uint32_t (&codes)[4], uint32_t &byte)
{
    float x[16];
    float amax = 0.0f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 f = unpack_16x2<kBf16>(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
        finite = finite && fabsf(f.x) <= 3.402823466e38f && fabsf(f.y) <= 3.402823466e38f; // false for NaN and infinities
        amax = fmaxf(amax, fmaxf(fabsf(f.x), fabsf(f.y)));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    const uint32_t vote = __ballot_sync(0xffffffffu, finite);
    finite = ((vote >> (lane_id() & 30u)) & 3u) == 3u;
    byte = finite ? mx_scale_byte(amax, kFmt == kKvMxFp4) : 255u;
    const float inv = mx_inverse_scale(finite ? byte : 127u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kFmt == kKvMxFp8) {
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] * inv, x[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] * inv, x[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
            codes[i] = lo | (hi << 16);
        } else {
            const uint32_t lo = __nv_cvt_float2_to_fp4x2(make_float2(x[4 * i] * inv, x[4 * i + 1] * inv), __NV_E2M1, cudaRoundNearest);
            const uint32_t hi = __nv_cvt_float2_to_fp4x2(make_float2(x[4 * i + 2] * inv, x[4 * i + 3] * inv), __NV_E2M1, cudaRoundNearest);
            codes[i] = lo | (hi << 8);
        }
        codes[i] = finite ? codes[i] : 0u;
    }
}

struct WriteArgs {
    const uint16_t *src[2];   // K, V: (tokens, kv_heads, d) with strides
    int64_t token_stride[2], head_stride[2];
    uint8_t *data[2];
    uint8_t *scale[2];
    const int32_t *slots;
    int64_t items; // tokens * kv_heads * (d / 16)
    int64_t num_slots;
    int kv_heads, page_shift, d;
};

// one thread: 16 elements of one token's head, of K (blockIdx.y 0) or V (1).  Lanes of a pair stay together: the
// number of threads a row takes (d / 16) is even.
template <bool kBf16, int kFmt>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const __grid_constant__ WriteArgs a, DeviceStatus *status)
{
    const int which = blockIdx.y;
    const int part_bits = a.d == 128 ? 3 : 2;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const bool in_range = idx < a.items;
    const uint32_t row = in_range ? static_cast<uint32_t>(idx >> part_bits) : 0u; // fewer than 2^31
    const int part = static_cast<int>(idx) & ((1 << part_bits) - 1);
    const uint32_t token = row / static_cast<uint32_t>(a.kv_heads);
    const int head = static_cast<int>(row - token * static_cast<uint32_t>(a.kv_heads));
    const int64_t slot = in_range ? a.slots[token] : -1;
    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (in_range) { // rows without a slot too: the load does not wait for the slot
        const uint16_t *src = a.src[which] + token * a.token_stride[which] + head * a.head_stride[which] + part * kPer;
        const int4 lo = ld_stream_i4(reinterpret_cast<const int4 *>(src));
        const int4 hi = ld_stream_i4(reinterpret_cast<const int4 *>(src) + 1);
        w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w;
        w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
    }
    bool live = slot >= 0;
    if (live && slot >= a.num_slots) {
        live = false;
        report_index(status, 10, static_cast<int>(slot));
    }
    // row of the cache: ((page * kv_heads + head) << page_shift) + position within the page
    const int64_t page = slot >> a.page_shift;
    const int64_t at = (((page * a.kv_heads + head) << a.page_shift) + (slot & ((1 << a.page_shift) - 1)));
    if constexpr (kFmt <= kKvBf16) {
        if (live) {
            uint4 *dst = reinterpret_cast<uint4 *>(a.data[which] + at * (2 * a.d) + part * 32);
            dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
            dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    } else {
        uint32_t codes[4], byte;
        encode16<kBf16, kFmt>(w, codes, byte);
        if (live) {
            if constexpr (kFmt == kKvMxFp8) {
                *reinterpret_cast<uint4 *>(a.data[which] + at * a.d + part * 16) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
            } else {
                *reinterpret_cast<uint2 *>(a.data[which] + at * (a.d / 2) + part * 8) =
                    make_uint2(codes[0] | (codes[1] << 16), codes[2] | (codes[3] << 16));
            }
            if ((part & 1) == 0) {
                a.scale[which][at * (a.d / 32) + part / 2] = static_cast<uint8_t>(byte);
            }
        }
    }
}

struct ReadArgs {
    const uint8_t *data[2];
    const uint8_t *scale[2];
    uint16_t *dst[2]; // (batch, kv_heads, max_len, d)
    const int32_t *table;
    const int32_t *lens;
    int64_t table_stride;
    int64_t num_pages;
    int table_cols, batch, kv_heads, max_len, page_shift, d;
};

// A thread makes 8 elements (16 bytes) of kRows tokens of one head, of K and of V, and has the loads of all of them under way
// before it converts the first: page table, then codes and scales, then stores are three waits a block, not three a row.
template <bool kBf16, int kFmt>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadArgs a, DeviceStatus *status)
{
    constexpr int kRows = kReadRows;
    constexpr bool k16 = kFmt <= kKvBf16;
    constexpr int kWords = k16 ? 4 : (kFmt == kKvMxFp8 ? 2 : 1); // of 8 elements in the cache
    const int part_bits = a.d == 128 ? 4 : 3;
    const int part = threadIdx.x & ((1 << part_bits) - 1);
    const int step = kThreads >> part_bits; // tokens between a thread's rows
    const int t0 = static_cast<int>(blockIdx.x) * (step * kRows) + (threadIdx.x >> part_bits);
    for (int64_t bh = blockIdx.y; bh < static_cast<int64_t>(a.batch) * a.kv_heads; bh += gridDim.y) {
        const int b = static_cast<int>(static_cast<uint32_t>(bh) / static_cast<uint32_t>(a.kv_heads));
        const int head = static_cast<int>(bh - static_cast<int64_t>(b) * a.kv_heads);
        const int len = min(a.lens[b], a.max_len);
        int64_t at[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int t = t0 + r * step, col = t >> a.page_shift;
            at[r] = -1;
            if (t < len) {
                const int64_t page = col < a.table_cols ? a.table[b * a.table_stride + col] : -1;
                if (page < 0 || page >= a.num_pages) {
                    report_index(status, 11, static_cast<int>(page));
                } else {
                    at[r] = ((page * a.kv_heads + head) << a.page_shift) + (t & ((1 << a.page_shift) - 1));
                }
            }
        }
        uint32_t w[2][kRows][kWords], byte[2][kRows];
#pragma unroll
        for (int which = 0; which < 2; ++which) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    w[which][r][i] = 0;
                }
                byte[which][r] = 127;
                if (at[r] >= 0) {
                    // rows of the cache are kWords 4-byte words times the threads of a row
                    const uint8_t *src = a.data[which] + ((at[r] << part_bits) + part) * (kWords * 4);
                    uint32_t *to = w[which][r];
                    if constexpr (kWords == 4) {
                        const int4 v = ld_stream_i4(reinterpret_cast<const int4 *>(src));
                        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
                    } else if constexpr (kWords == 2) {
                        const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(src));
                        to[0] = v.x, to[1] = v.y;
                    } else {
                        to[0] = __ldcs(reinterpret_cast<const unsigned *>(src));
                    }
                    if constexpr (!k16) { // four threads a scale
                        byte[which][r] = a.scale[which][((at[r] << part_bits) + part) >> 2];
                    }
                }
            }
        }
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            uint16_t *dst = a.dst[which] + (bh * a.max_len + t0) * a.d + part * 8;
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                uint32_t out[4];
                const uint32_t *from = w[which][r];
                if constexpr (k16) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        out[i] = from[i];
                        if constexpr ((kFmt == kKvBf16) != kBf16) { // a cache of the other 16-bit type: one rounding
                            const float2 f = unpack_16x2<kFmt == kKvBf16>(out[i]);
                            out[i] = pack_16x2<kBf16>(f.x, f.y);
                        }
                    }
                } else {
                    uint32_t h[4];
                    if constexpr (kFmt == kKvMxFp8) {
                        e4m3x4_to_f16(from[0], h[0], h[1]);
                        e4m3x4_to_f16(from[1], h[2], h[3]);
                    } else {
                        e2m1x8_to_f16(from[0], h);
                    }
                    const float s = e8m0x2_to_f32(byte[which][r]).x;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = unpack_16x2<false>(h[i]);
                        out[i] = pack_16x2<kBf16>(f.x * s, f.y * s);
                    }
                }
                if (t0 + r * step < a.max_len) {
                    st_stream_u4(reinterpret_cast<uint4 *>(dst + static_cast<int64_t>(r * step) * a.d), make_uint4(out[0], out[1], out[2], out[3]));
                }
            }
        }
    }
}

} // namespace

int launch_kv_write(const KvCacheView &cache, const uint16_t *k, const uint16_t *v, bool bf16, const int32_t *slots,
                    int64_t tokens, const int64_t strides[4], cudaStream_t stream)
{
    DeviceStatus *status = device_status_ptr();
    if (status == nullptr) {
        return kErrCuda;
    }
    WriteArgs a;
    a.src[0] = k;
    a.src[1] = v;
    a.token_stride[0] = strides[0];
    a.head_stride[0] = strides[1];
    a.token_stride[1] = strides[2];
    a.head_stride[1] = strides[3];
    a.data[0] = static_cast<uint8_t *>(cache.k);
    a.data[1] = static_cast<uint8_t *>(cache.v);
    a.scale[0] = cache.k_scale;
    a.scale[1] = cache.v_scale;
    a.slots = slots;
    a.items = tokens * cache.kv_heads * (cache.d / kPer);
    a.num_slots = cache.num_pages << cache.page_shift;
    a.kv_heads = cache.kv_heads;
    a.page_shift = cache.page_shift;
    a.d = cache.d;
    const int64_t blocks = (a.items + kThreads - 1) / kThreads;
    if (tokens * cache.kv_heads > 0x7fffffffLL) {
        set_error_text("kv_cache_write: too many rows for one call");
        return kErrTooLarge;
    }
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    switch (cache.fmt) {
        case kKvF16:
        case kKvBf16: kv_write_kernel<false, kKvF16><<<grid, kThreads, 0, stream>>>(a, status); break;
        case kKvMxFp8:
            bf16 ? kv_write_kernel<true, kKvMxFp8><<<grid, kThreads, 0, stream>>>(a, status)
                 : kv_write_kernel<false, kKvMxFp8><<<grid, kThreads, 0, stream>>>(a, status);
            break;
        default:
            bf16 ? kv_write_kernel<true, kKvMxFp4><<<grid, kThreads, 0, stream>>>(a, status)
                 : kv_write_kernel<false, kKvMxFp4><<<grid, kThreads, 0, stream>>>(a, status);
    }
    return check_launch();
}

int launch_kv_read(const KvCacheView &cache, const int32_t *table, int64_t table_stride, int table_cols,
                   const int32_t *lens, int batch, int max_len, uint16_t *k, uint16_t *v, bool bf16, cudaStream_t stream)
{
    DeviceStatus *status = device_status_ptr();
    if (status == nullptr) {
        return kErrCuda;
    }
    ReadArgs a;
    a.data[0] = static_cast<const uint8_t *>(cache.k);
    a.data[1] = static_cast<const uint8_t *>(cache.v);
    a.scale[0] = cache.k_scale;
    a.scale[1] = cache.v_scale;
    a.dst[0] = k;
    a.dst[1] = v;
    a.table = table;
    a.lens = lens;
    a.table_stride = table_stride;
    a.num_pages = cache.num_pages;
    a.table_cols = table_cols;
    a.batch = batch;
    a.kv_heads = cache.kv_heads;
    a.max_len = max_len;
    a.page_shift = cache.page_shift;
    a.d = cache.d;
    const int64_t heads = static_cast<int64_t>(batch) * cache.kv_heads;
    const int tokens = kThreads / (cache.d / 8) * kReadRows; // of a block
    const dim3 grid(static_cast<unsigned>((max_len + tokens - 1) / tokens),
                    static_cast<unsigned>(heads < 65535 ? heads : 65535));
#define PTO_B200_KV_READ(fmt)                                              \
    bf16 ? kv_read_kernel<true, fmt><<<grid, kThreads, 0, stream>>>(a, status) \
         : kv_read_kernel<false, fmt><<<grid, kThreads, 0, stream>>>(a, status)
    switch (cache.fmt) {
        case kKvF16: PTO_B200_KV_READ(kKvF16); break;
        case kKvBf16: PTO_B200_KV_READ(kKvBf16); break;
        case kKvMxFp8: PTO_B200_KV_READ(kKvMxFp8); break;
        default: PTO_B200_KV_READ(kKvMxFp4);
    }
#undef PTO_B200_KV_READ
    return check_launch();
}

} // namespace pto_b200
