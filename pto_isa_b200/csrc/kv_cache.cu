// The paged key / value cache: rows are quantised as they are written and read back as 16-bit tensors.
//
// A cache holds K and V as (pages, kv_heads, page_size, row) with a row of head_dim elements in 16 bits, in MX fp8
// (float8_e4m3fn) or MX fp4 (float4_e2m1, the lower index in the low nibble), the MX formats with one e8m0 scale byte per
// 32 elements in (pages, kv_heads, page_size, head_dim / 32).  For a block x of 32 elements
//     a = max |x|,  e = the smallest integer with a <= M 2^e (M = 448 or 6),  code = RNE(x 2^-e),  value = code 2^e:
// everything but the one rounding is exact, so a row's codes do not depend on who computes them.  A block that holds a
// NaN or an infinity gets the scale byte 255 and reads back as NaN throughout (e2m1 has no NaN of its own).
//
// Both kernels move bytes and are bound by HBM: a thread owns 16 elements (32 bytes of the 16-bit side, half a scale
// block: its partner is one lane away), so every access is 16 bytes wide or, for fp4 codes, 8.
#include "ptx.cuh"
#include "internal.h"
#include "mx_format.cuh"

namespace pto_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16; // elements a thread owns

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
    const int parts = a.d / kPer;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    const bool in_range = idx < a.items;
    const int64_t row = in_range ? idx / parts : 0;
    const int part = static_cast<int>(idx % parts);
    const int64_t token = row / a.kv_heads;
    const int head = static_cast<int>(row % a.kv_heads);
    const int64_t slot = in_range ? a.slots[token] : -1;
    bool live = slot >= 0;
    if (live && slot >= a.num_slots) {
        live = false;
        report_index(status, 10, static_cast<int>(slot));
    }
    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (live) {
        const uint16_t *src = a.src[which] + token * a.token_stride[which] + head * a.head_stride[which] + part * kPer;
        const int4 lo = ld_stream_i4(reinterpret_cast<const int4 *>(src));
        const int4 hi = ld_stream_i4(reinterpret_cast<const int4 *>(src) + 1);
        w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w;
        w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
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
    int64_t row_items; // max_len * (d / 16)
    int table_cols, batch, kv_heads, max_len, page_shift, d;
};

template <bool kBf16, int kFmt>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const __grid_constant__ ReadArgs a, DeviceStatus *status)
{
    const int parts = a.d / kPer;
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if (idx >= a.row_items) {
        return;
    }
    const int t = static_cast<int>(idx / parts);
    const int part = static_cast<int>(idx % parts);
    for (int64_t bh = blockIdx.y; bh < static_cast<int64_t>(a.batch) * a.kv_heads; bh += gridDim.y) {
        const int b = static_cast<int>(bh / a.kv_heads), head = static_cast<int>(bh % a.kv_heads);
        uint32_t out[2][8];
#pragma unroll
        for (int which = 0; which < 2; ++which) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                out[which][i] = 0u;
            }
        }
        if (t < a.lens[b]) {
            const int col = t >> a.page_shift;
            const int64_t page = col < a.table_cols ? a.table[b * a.table_stride + col] : -1;
            if (page < 0 || page >= a.num_pages) {
                report_index(status, 11, static_cast<int>(page));
            } else {
                const int64_t at = ((page * a.kv_heads + head) << a.page_shift) + (t & ((1 << a.page_shift) - 1));
#pragma unroll
                for (int which = 0; which < 2; ++which) {
                    if constexpr (kFmt <= kKvBf16) {
                        const int4 *src = reinterpret_cast<const int4 *>(a.data[which] + at * (2 * a.d) + part * 32);
                        const int4 lo = ld_stream_i4(src), hi = ld_stream_i4(src + 1);
                        const int w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if constexpr ((kFmt == kKvBf16) == kBf16) {
                                out[which][i] = w[i];
                            } else { // a cache of the other 16-bit type: one rounding
                                const float2 f = unpack_16x2<kFmt == kKvBf16>(w[i]);
                                out[which][i] = pack_16x2<kBf16>(f.x, f.y);
                            }
                        }
                    } else {
                        const float s = e8m0_value(a.scale[which][at * (a.d / 32) + part / 2]);
                        uint32_t h[8];
                        if constexpr (kFmt == kKvMxFp8) {
                            const int4 c = ld_stream_i4(reinterpret_cast<const int4 *>(a.data[which] + at * a.d + part * 16));
                            const uint32_t w[4] = {static_cast<uint32_t>(c.x), static_cast<uint32_t>(c.y),
                                                   static_cast<uint32_t>(c.z), static_cast<uint32_t>(c.w)};
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                h[i] = e4m3x2_to_f16x2((w[i >> 1] >> ((i & 1) * 16)) & 0xffffu);
                            }
                        } else {
                            const uint2 c = *reinterpret_cast<const uint2 *>(a.data[which] + at * (a.d / 2) + part * 8);
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                h[i] = e2m1x2_to_f16x2(((i < 4 ? c.x : c.y) >> ((i & 3) * 8)) & 0xffu);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float2 f = unpack_16x2<false>(h[i]);
                            out[which][i] = pack_16x2<kBf16>(f.x * s, f.y * s);
                        }
                    }
                }
            }
        }
        const int64_t to = (bh * a.max_len + t) * a.d + part * kPer;
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            uint4 *dst = reinterpret_cast<uint4 *>(a.dst[which] + to);
            st_stream_u4(dst, make_uint4(out[which][0], out[which][1], out[which][2], out[which][3]));
            st_stream_u4(dst + 1, make_uint4(out[which][4], out[which][5], out[which][6], out[which][7]));
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
    if (blocks > 0x7fffffffLL) {
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
    a.row_items = static_cast<int64_t>(max_len) * (cache.d / kPer);
    a.table_cols = table_cols;
    a.batch = batch;
    a.kv_heads = cache.kv_heads;
    a.max_len = max_len;
    a.page_shift = cache.page_shift;
    a.d = cache.d;
    const int64_t heads = static_cast<int64_t>(batch) * cache.kv_heads;
    const dim3 grid(static_cast<unsigned>((a.row_items + kThreads - 1) / kThreads),
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
