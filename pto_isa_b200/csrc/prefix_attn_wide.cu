// The shared prefix's keys against many query rows, on the fifth-generation tensor cores (the part of prefix_attn whose
// rows are those of the whole batch; prefix_attn.cu says how the parts are joined).
//
// One block per SM takes 128-row tiles of one kv head's rows (all sequences, query tokens and heads of the group) and a run
// of the prefix's keys, 128 at a time:
//   S = Q K^T   tcgen05.mma, both operands K-major in 128-byte-swizzled shared memory, S in tensor memory
//   softmax     one thread per row: running maximum and sum in registers, P in 16 bits to shared memory
//   O += P V    tcgen05.mma, V MN-major (as its rows lie), O in tensor memory, rescaled only when a row's maximum has
//               grown 256-fold
// and leaves (O, m, l) in fp32.  Two groups of four softmax warps: with more than one tile of rows they take two tiles and
// share every K and V tile (kPair), with a single tile they take alternate key tiles, so that one group's exponentials
// run under the other's products either way.
//
// A tile of K or V comes from pages, in 16 bits by cp.async or as codes that eight loading warps convert on the way into
// shared memory.  Codes become float16 whatever the type of q: e4m3 and e2m1 convert to float16 pairs in one instruction,
// to bfloat16 in four.  Exactness:
//   K       code 2^e is exact in float16 for e in [-15, 7] (e4m3) or [-23, 13] (e2m1).  A key with a block outside that range is
//           stored relative to its largest scale, 2^(e - e_max), and the power of two goes to the logit as a factor of the key
//           (NaN where a scale byte is 255).  Blocks far below the key's largest then lose bits: at most 2^-25 2^(e_max) an
//           element.
//   q       bfloat16 rows are divided by a power of two that brings their largest element into [2^14, 2^15): elements
//           down to 2^-31 of it keep every bit; the logits of the row are multiplied back.
//   V, P    float16 where all scales of the tile are in range; otherwise, if q is bfloat16, this tile's V and P are bfloat16
//           (code 2^e is exact there): an instruction's operands share a type, its fp32 accumulator does not care.  If q is
//           float16 V is rounded to float16, which takes scales of 2^-24 to 2^15 or a tile made by way of 32 bits.  A block of
//           scale byte 0 counts as out of range, of K as well: whether it is all zeros would take its codes (looked up by the
//           describing warps, 8 x 128 rows x 32768 MX fp4 keys without any such block took 6 us more).
//
// What bounds it: per 128 x 128 logits and head size 128, 1024 cycles of tensor work, 1024 of the special-function unit
// (an exponential takes 8 cycles a warp), about 512 of the integer pipe for the conversion of a quantised tile.  It takes
// 4200 for a softmax group and about 4000 for a quantised tile's loaders (a tile's loads, conversion, fence and hand-over one
// after another), and 9 to 10 thousand before the first product: 8 heads x 512 rows x 8192 float16 keys 41 us, 8 x 128 rows x
// 32768 MX fp4 keys 47 us (68 thousand cycles for 15 key tiles a block).  A tile's loaders wait for its description, so what that
// takes counts: with a row's scale bytes compared one by one the latter took 4 us more.
#include "ptx.cuh"
#include "prefix_attn.cuh"

namespace pto_b200 {

namespace {

constexpr int kThreads = 640; // warps 0-3, 4-7 softmax; 8-11 loading K, 12-15 loading V; 16, 17 issuing (one per group); 18, 19
// describing the key tiles and fetching them towards L2
// registers of a thread: 96 at launch (five warps a scheduler), then 2 * 112 + 2 * 80 + 96, times 128, which is all of these
// 640 * 96.  No role may spill: shared memory leaves the first-level cache so little that every reload comes from L2 (with 40
// registers the issuing threads reloaded descriptors and took 700 cycles for a product).  Over MX caches of head size 128 some
// forms do, one to five registers.
constexpr int kRegsLaunch = 96, kRegsSoftmax = 112, kRegsLoad = 80, kRegsIssue = 96;
static_assert((2 * kRegsSoftmax + 2 * kRegsLoad + kRegsIssue) * 128 <= kThreads * kRegsLaunch, "an increase would wait forever");
constexpr int kIssueWarp = 16;
constexpr int kTile = 128;
constexpr int kTmemCols = 512;
constexpr float kDefer = 8.0f; // log2 of the growth of a row's maximum that rescales O

struct Info { // of a key tile
    uint32_t valid[4]; // bit r: key r exists
    uint32_t flags[4]; // by 32 keys: bit 0, some key has a factor; bit 1, V by way of 32 bits, to bfloat16 if q is
    uint16_t factor[kTile]; // bfloat16, a power of two
};

template <int kD, bool kPair>
struct Shape {
    static constexpr int kTileBytes = kTile * kD * 2; // Q, K, V
    static constexpr int kHalfBytes = kTile * 128;    // 64 columns of 16 bits, one swizzled half
    static constexpr int kPBytes = 2 * kHalfBytes;
    static constexpr int kQTiles = kPair ? 2 : 1;
    static constexpr int kRingK = kD == 64 ? 3 : 2, kRingV = kD == 64 ? 3 : (kPair ? 1 : 2);
    // Tiles whose description is kept.  Tile m + 1 is described when K(m) has been stored, so when the product with
    // K(m - kRingK) is complete; the oldest tile that a group can then still be at is m - 6 (one tile of rows, three slots:
    // the group of K(m - 4) has yet to issue the product with V(m - 6)).
    static constexpr int kInfo = 8;
    struct Control {
        uint64_t q_full[2];
        uint64_t k_full[kRingK], k_empty[kRingK], v_full[kRingV], v_empty[kRingV];
        uint64_t info_full[kInfo];
        uint64_t s_full[2], s_free[2], p_full[2], pv_done[2];
        uint32_t tmem_base;
        int abort_flag;
        float q_factor[kPair ? 1 : kTile]; // what the rows of q were divided by, for the group that did not load them
        Info info[kInfo];
    };
    static constexpr int kData = (kQTiles + kRingK + kRingV) * kTileBytes + 2 * kPBytes;
    static constexpr int kSmem = kData + static_cast<int>(sizeof(Control));
    static_assert(kSmem <= 232448, "shared memory of a block");
};

__device__ __forceinline__ float ex2w(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// a whole warp waits: one lane polls, what it has acquired holds for the warp
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int lane)
{
    bool ok = true;
    if (lane == 0) {
        ok = mbar_wait(bar, parity, abort_flag);
    }
    return __shfl_sync(0xffffffffu, ok, 0);
}

// where 16 bytes (8 elements) `chunk` of row `row` lie in a 64-column half
__device__ __forceinline__ uint32_t swz(int row, int chunk)
{
    return static_cast<uint32_t>(row * 128 + ((chunk ^ (row & 7)) << 4));
}

// the scale bytes of a row: d / 32 of them
template <int kD>
__device__ __forceinline__ uint32_t row_scales(const uint8_t *s, int64_t row)
{
    if constexpr (kD == 128) {
        return __ldg(reinterpret_cast<const uint32_t *>(s) + row);
    } else {
        return __ldg(reinterpret_cast<const uint16_t *>(s) + row);
    }
}

// whether all scale bytes of a row lie in [kLow, kHigh]: four subtractions side by side.  A byte below kLow borrows, but has bit 7
// itself then, and only bytes above it see the borrow.
template <int kD, uint32_t kLow, uint32_t kHigh>
__device__ __forceinline__ bool bytes_within(uint32_t s)
{
    static_assert(kLow <= kHigh && kLow + 128 > kHigh && 255 - kLow + 127 - (kHigh - kLow) < 256, "a sum would carry");
    const uint32_t x = s - kLow * 0x01010101u;
    return (((x + (127 - (kHigh - kLow)) * 0x01010101u) | x) & (kD == 64 ? 0x8080u : 0x80808080u)) == 0;
}

// Whether code 2^(byte - 127) is exact in float16 for every block of the row: e in [-15, 7] for e4m3 (2^-9 .. 448), in
// [-23, 13] for e2m1 (0.5 .. 6).  Byte 0 is not among them: it mostly stands for zeros, but may be multiples of 2^-127.
template <int kD, int kFmt>
__device__ __forceinline__ bool scales_in_range(uint32_t s)
{
    return kFmt == kKvMxFp8 ? bytes_within<kD, 112, 134>(s) : bytes_within<kD, 104, 140>(s);
}

// whether one float16 product makes a row of V: for bfloat16 queries with every bit, for float16 queries rounded to float16, which
// takes powers of two that it has, 2^-24 to 2^15
template <bool kBf16, int kD, int kFmt>
__device__ __forceinline__ bool value_is_plain(uint32_t s)
{
    return kBf16 ? scales_in_range<kD, kFmt>(s) : bytes_within<kD, 103, 142>(s);
}

template <int kD>
__device__ __forceinline__ uint32_t largest_scale(uint32_t s)
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kD / 32; ++i) {
        m = max(m, (s >> (8 * i)) & 0xffu);
    }
    return m;
}

// sixteen codes -> sixteen float16 (8 words)
template <int kFmt>
__device__ __forceinline__ void codes16_to_f16(const uint32_t *c, uint32_t (&h)[8])
{
    if constexpr (kFmt == kKvMxFp8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e4m3x4_to_f16(c[i], h[2 * i], h[2 * i + 1]);
        }
    } else {
        e2m1x8_to_f16(c[0], *reinterpret_cast<uint32_t(*)[4]>(h));
        e2m1x8_to_f16(c[1], *reinterpret_cast<uint32_t(*)[4]>(h + 4));
    }
}

template <bool kBf16, int kD, int kFmt, bool kPair>
__global__ void __launch_bounds__(kThreads, 1) prefix_wide_kernel(const __grid_constant__ AttnArgs a, DeviceStatus *status)
{
    using Sh = Shape<kD, kPair>;
    using Control = typename Sh::Control;
    constexpr bool kMx = kFmt >= kKvMxFp8;
    constexpr bool kOpBf16 = kBf16 && !kMx; // type of the products' operands (but for V and P of flagged tiles)
    constexpr int kRingK = Sh::kRingK, kRingV = Sh::kRingV, kInfo = Sh::kInfo;
    constexpr int kHalves = kD / 64;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint8_t *smem_q = smem;
    uint8_t *smem_k = smem_q + Sh::kQTiles * Sh::kTileBytes;
    uint8_t *smem_v = smem_k + kRingK * Sh::kTileBytes;
    uint8_t *smem_p = smem_v + kRingV * Sh::kTileBytes;
    Control *ctl = reinterpret_cast<Control *>(smem_p + 2 * Sh::kPBytes);

    programmatic_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- which rows and keys: block = ((split * kv_heads) + h) * row blocks + row block
    const int rows = a.batch * a.tokens * a.group;
    const int row_blocks = (rows + kTile * Sh::kQTiles - 1) / (kTile * Sh::kQTiles);
    const int rb = blockIdx.x % row_blocks;
    const int h = blockIdx.x / row_blocks % a.kv_heads;
    const int split = blockIdx.x / row_blocks / a.kv_heads;
    const int k_begin = split * a.prefix_chunk;
    const int k_end = min(k_begin + a.prefix_chunk, a.prefix_len);
    const int tiles = (k_end - k_begin + kTile - 1) / kTile;
    // group t: pair form, row tile 2 rb + t and every key tile; single form, row tile rb and key tiles t, t + 2, ..
    const bool group_rows[2] = {true, kPair ? (2 * rb + 1) * kTile < rows : true};

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&ctl->q_full[t], 4);
            mbar_init(&ctl->s_full[t], 1);
            mbar_init(&ctl->s_free[t], 4);
            mbar_init(&ctl->p_full[t], 4);
            mbar_init(&ctl->pv_done[t], 1);
        }
        for (int s = 0; s < kRingK; ++s) {
            mbar_init(&ctl->k_full[s], 4);
            mbar_init(&ctl->k_empty[s], kPair ? 2 : 1);
        }
        for (int s = 0; s < kRingV; ++s) {
            mbar_init(&ctl->v_full[s], 4);
            mbar_init(&ctl->v_empty[s], kPair ? 2 : 1);
        }
        for (int s = 0; s < kInfo; ++s) {
            mbar_init(&ctl->info_full[s], 2);
        }
        ctl->abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == kIssueWarp) {
        tmem_alloc(&ctl->tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = ctl->tmem_base;
    volatile int *abort_flag = &ctl->abort_flag;
    constexpr int RB = kv_row_bytes(kFmt, kD);
    const int page_mask = (1 << a.page_shift) - 1;
    // page of key r of tile j; -1: no such key.  Numbers out of range count as if there were no key.
    auto page_of = [&](int j, int r) -> int {
        const int key = k_begin + j * kTile + r;
        return key < k_end ? __ldg(a.prefix_pages + (key >> a.page_shift)) : -1;
    };
    // row of the cache of key r of tile j, which lies in `page`; -1 for none
    auto cache_row = [&](int page, int j, int r) -> int64_t {
        return page < 0 || page >= a.num_pages
                   ? -1
                   : ((static_cast<int64_t>(page) * a.kv_heads + h) << a.page_shift) + ((k_begin + j * kTile + r) & page_mask);
    };

    if (warp >= kIssueWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
        // ------------------------------------------------------------ issuing warps, one per group
        const int t = warp - kIssueWarp;
        if (t < 2 && lane == 0) {
            constexpr uint32_t idesc_s = make_idesc_f16(kTile, kTile, 0, 0, kOpBf16 ? 1 : 0);
            constexpr uint32_t idesc_o = make_idesc_f16(kTile, kD, 0, 1, kOpBf16 ? 1 : 0);
            constexpr uint32_t idesc_ob = make_idesc_f16(kTile, kD, 0, 1, 1);
            const uint32_t s_tmem = tmem_base + t * 128, o_tmem = tmem_base + 256 + t * 128;
            const uint64_t q_desc = make_sw128_desc(smem_u32(smem_q) + (kPair ? t : 0) * Sh::kTileBytes, 16, 1024);
            const uint64_t p_desc = make_sw128_desc(smem_u32(smem_p) + t * Sh::kPBytes, 16, 1024);
            auto kstep = [](int kk) -> uint64_t { return static_cast<uint64_t>((kk >> 2) * (Sh::kHalfBytes >> 4) + (kk & 3) * 2); };
            bool ok = true;
            // S of the group's n-th tile (key tile j)
            auto do_s = [&](int j, int n) {
                const int slot = j % kRingK;
                const uint32_t addr = smem_u32(smem_k) + slot * Sh::kTileBytes;
                ok = mbar_wait(&ctl->k_full[slot], (j / kRingK) & 1, abort_flag);
                if (ok && group_rows[t]) {
                    if (n == 0) {
                        ok = mbar_wait(&ctl->q_full[kPair ? t : 0], 0, abort_flag);
                    } else {
                        ok = mbar_wait(&ctl->s_free[t], (n - 1) & 1, abort_flag); // the previous S has been read
                    }
                    if (ok) {
                        tc_fence_after();
                        const uint64_t k_desc = make_sw128_desc(addr, 16, 1024);
#pragma unroll
                        for (int kk = 0; kk < kD / 16; ++kk) {
                            tc_mma_f16_ss(s_tmem, q_desc + kstep(kk), k_desc + kstep(kk), idesc_s, kk != 0 ? 1u : 0u);
                        }
                        tc_commit(&ctl->s_full[t]);
                    }
                }
                if (ok) {
                    tc_commit(&ctl->k_empty[slot]);
                }
            };
            auto do_pv = [&](int j, int n) {
                const int slot = j % kRingV;
                const uint32_t addr = smem_u32(smem_v) + slot * Sh::kTileBytes;
                ok = mbar_wait(&ctl->v_full[slot], (j / kRingV) & 1, abort_flag);
                if (ok && group_rows[t]) {
                    ok = mbar_wait(&ctl->p_full[t], n & 1, abort_flag);
                    if (ok) {
                        tc_fence_after();
                        uint32_t idesc = idesc_o;
                        if constexpr (kMx && kBf16) {
                            const Info &info = ctl->info[j % kInfo];
                            const uint32_t f = info.flags[0] | info.flags[1] | info.flags[2] | info.flags[3];
                            idesc = (f & 2u) ? idesc_ob : idesc_o;
                        }
                        const uint64_t v_desc = make_sw128_desc(addr, Sh::kHalfBytes, 1024); // MN-major: 16 keys = 2 KiB
#pragma unroll
                        for (int kk = 0; kk < kTile / 16; ++kk) {
                            tc_mma_f16_ss(o_tmem, p_desc + kstep(kk), v_desc + static_cast<uint64_t>(kk * 128), idesc,
                                          (n != 0 || kk != 0) ? 1u : 0u);
                        }
                        tc_commit(&ctl->pv_done[t]);
                    }
                }
                if (ok) {
                    tc_commit(&ctl->v_empty[slot]);
                }
            };
            // S of a tile is issued before the product with V of the one before it
            constexpr int kHop = kPair ? 1 : 2;
            int n = -1;
#pragma unroll 1
            for (int j = (kPair ? 0 : t) - kHop; j < tiles && ok; j += kHop, ++n) {
                if (j + kHop < tiles) {
                    do_s(j + kHop, n + 1);
                }
                if (ok && n >= 0) {
                    do_pv(j, n);
                }
            }
        } else if (t >= 2) {
            // -------------------------------------------------------- describing warps: two keys a thread.  Page numbers and
            // scales are loaded a tile ahead; tile m follows when K(m - 1) has been stored.
            const int r = (t - 2) * 32 + lane;
            int pid[2], pid_next[2];
            uint32_t ks[2] = {0, 0}, vs[2] = {0, 0};
            auto load_scales = [&](int m) {
#pragma unroll
                for (int i = 0; i < 2 && kMx; ++i) {
                    const int64_t row = cache_row(pid[i], m, r + 64 * i);
                    ks[i] = row >= 0 ? row_scales<kD>(a.ks, row) : 0x7f7f7f7fu; // no key: nothing out of the ordinary
                    vs[i] = row >= 0 ? row_scales<kD>(a.vs, row) : 0x7f7f7f7fu;
                }
            };
            // 16 keys a lane: K by one warp, V by the other
            auto fetch = [&](int page, int m, int lane8) {
                const int64_t row = m < tiles ? cache_row(page, m, lane8 * 16) : -1;
                if (row >= 0) {
                    const uint8_t *src = (t == 2 ? a.k : a.v) + row * RB;
                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(16 * RB) : "memory");
                }
            };
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                pid[i] = page_of(0, r + 64 * i);
                pid_next[i] = tiles > 1 ? page_of(1, r + 64 * i) : -1;
            }
            int pid_l2 = tiles > 3 && lane < 8 ? page_of(3, lane * 16) : -1;
            if (lane < 16) { // tiles 1 and 2 at once
                const int m = 1 + (lane >> 3);
                fetch(m < tiles ? page_of(m, (lane & 7) * 16) : -1, m, lane & 7);
            }
            load_scales(0);
#pragma unroll 1
            for (int m = 0; m < tiles; ++m) {
                if (m > 0 && !warp_wait(&ctl->k_full[(m - 1) % kRingK], ((m - 1) / kRingK) & 1, abort_flag, lane)) {
                    break;
                }
                Info &info = ctl->info[m % kInfo];
                uint32_t valid[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    valid[i] = __ballot_sync(0xffffffffu, pid[i] >= 0 && pid[i] < a.num_pages);
                    uint32_t flags = 0;
                    if constexpr (kMx) {
                        const bool k_out = !scales_in_range<kD, kFmt>(ks[i]);
                        const bool v_out = !value_is_plain<kBf16, kD, kFmt>(vs[i]);
                        const uint32_t top = largest_scale<kD>(ks[i]); // 255: NaN, whatever the block's codes are
                        info.factor[r + 64 * i] = k_out ? static_cast<uint16_t>(top == 255u ? 0x7fc0u : top == 0u ? 0x0040u : top << 7) : 0x3f80;
                        flags = (__any_sync(0xffffffffu, k_out) ? 1u : 0u) | (__any_sync(0xffffffffu, v_out) ? 2u : 0u);
                    }
                    if (lane == 0) {
                        info.valid[2 * i + t - 2] = valid[i];
                        info.flags[2 * i + t - 2] = flags;
                    }
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&ctl->info_full[m % kInfo]);
                }
                const int was[2] = {pid[0], pid[1]};
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    pid[i] = pid_next[i];
                    pid_next[i] = m + 2 < tiles ? page_of(m + 2, r + 64 * i) : -1;
                }
                load_scales(m + 1);
                if ((valid[0] & valid[1]) != 0xffffffffu) { // pages that do not exist: reported by one lane, when nobody waits for it
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t missing = __ballot_sync(0xffffffffu, k_begin + m * kTile + r + 64 * i < k_end) & ~valid[i];
                        if (missing != 0 && lane == __ffs(missing) - 1 && atomicCAS(&status->code, 0, kErrBadArgument) == 0) {
                            status->block = blockIdx.x;
                            status->where = 11;
                            status->detail = was[i];
                        }
                    }
                }
                if (lane < 8) {
                    fetch(pid_l2, m + 3, lane);
                    pid_l2 = m + 4 < tiles ? page_of(m + 4, lane * 16) : -1;
                }
            }
        }
    } else if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLoad));
        // ------------------------------------------------------------ loading warps
        // One warpgroup for K, one for V, the same code.  A thread's share of a tile: 16 elements p of each 64-column half in
        // the rows r0 + 32 i.  All loads of a tile are issued before any is used and the two groups take turns at waiting
        // for memory.  (Loads in flight across the fence before a hand-over would be waited for by it: no tile's loads are
        // issued before the last one has been handed over; the L2 prefetch, two tiles ahead, is what hides DRAM.)
        const bool is_v = warp >= 12;
        const int tid = threadIdx.x & 127;
        const int p = tid & 3, r0 = tid >> 2;
        const int ring = is_v ? kRingV : kRingK;
        uint64_t *full = is_v ? ctl->v_full : ctl->k_full, *empty = is_v ? ctl->v_empty : ctl->k_empty;
        const uint32_t ring_base = smem_u32(is_v ? smem_v : smem_k);
        const uint8_t *data = is_v ? a.v : a.k;
        const uint32_t at0 = swz(r0, 2 * p), at1 = at0 ^ 16; // of the two 16-byte chunks, row r0
        int pid[4]; // of this thread's rows in the next tile
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            pid[i] = page_of(0, r0 + 32 * i);
        }
        bool ok = true;
        int slot = 0;
        uint32_t phase = 1;
#pragma unroll 1
        for (int j = 0; j < tiles; ++j) {
            // ---- the tile's rows, and the pages of the next
            int64_t row[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                row[i] = cache_row(pid[i], j, r0 + 32 * i);
                pid[i] = j + 1 < tiles ? page_of(j + 1, r0 + 32 * i) : -1;
            }
            const uint32_t dst = ring_base + slot * Sh::kTileBytes;
            if constexpr (!kMx) {
                ok = warp_wait(&empty[slot], phase, abort_flag, lane);
                if (!ok) {
                    break;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint8_t *from = data + (row[i] < 0 ? 0 : row[i]) * RB + p * 32;
                    const int bytes = row[i] < 0 ? 0 : 16;
#pragma unroll
                    for (int half = 0; half < kHalves; ++half) {
                        const uint32_t to = dst + half * Sh::kHalfBytes + i * 32 * 128;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + at0), "l"(from + half * 128), "r"(bytes) : "memory");
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + at1), "l"(from + half * 128 + 16), "r"(bytes) : "memory");
                    }
                }
                asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
                // K is handed over when its tile has been described, as where its scales are needed: the describing warps, which
                // follow K's ring by its parity, are then never more than a round of it behind
                if (!is_v && !warp_wait(&ctl->info_full[j % kInfo], (j / kInfo) & 1, abort_flag, lane)) {
                    ok = false;
                    break;
                }
            } else {
                constexpr int kWords = kFmt == kKvMxFp8 ? 4 : 2;
                uint32_t code[4 * kHalves][kWords], scales[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool live = row[i] >= 0;
                    const uint8_t *src = data + row[i] * RB + p * (4 * kWords);
                    scales[i] = live ? row_scales<kD>(is_v ? a.vs : a.ks, row[i]) : 0u;
#pragma unroll
                    for (int half = 0; half < kHalves; ++half) {
                        uint32_t *c = code[i * kHalves + half];
                        if constexpr (kFmt == kKvMxFp8) {
                            const uint4 v = live ? __ldg(reinterpret_cast<const uint4 *>(src + half * 64)) : make_uint4(0, 0, 0, 0);
                            c[0] = v.x, c[1] = v.y, c[2] = v.z, c[3] = v.w;
                        } else {
                            const uint2 v = live ? __ldg(reinterpret_cast<const uint2 *>(src + half * 32)) : make_uint2(0, 0);
                            c[0] = v.x, c[1] = v.y;
                        }
                    }
                }
                ok = warp_wait(&empty[slot], phase, abort_flag, lane) &&
                     warp_wait(&ctl->info_full[j % kInfo], (j / kInfo) & 1, abort_flag, lane);
                if (!ok) {
                    break;
                }
                const Info &info = ctl->info[j % kInfo];
                const uint32_t flags = info.flags[0] | info.flags[1] | info.flags[2] | info.flags[3];
                const bool special = (flags & (is_v ? 2u : 1u)) != 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
#pragma unroll
                    for (int half = 0; half < kHalves; ++half) {
                        uint32_t w[8];
                        codes16_to_f16<kFmt>(code[i * kHalves + half], w);
                        // 2^(byte - 127) in both halves, where float16 has it: what it makes of others is made again below
                        const uint32_t byte = (scales[i] >> (8 * (half * 2 + (p >> 1)))) & 0xffu;
                        const float f = __uint_as_float(byte << 23);
                        const uint32_t m = pack_16x2<false>(f, f), to = dst + half * Sh::kHalfBytes + i * 32 * 128;
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            w[x] = mul_16x2<false>(w[x], m);
                        }
                        sts128(to + at0, w[0], w[1], w[2], w[3]);
                        sts128(to + at1, w[4], w[5], w[6], w[7]);
                    }
                }
                if (special) { // rare: the tile once more, from memory, in small steps
#pragma unroll 1
                    for (int u = 0; u < 4 * kHalves; ++u) {
                        const int i = u / kHalves, half = u % kHalves;
                        const int64_t at = cache_row(page_of(j, r0 + 32 * i), j, r0 + 32 * i);
                        uint32_t c[4] = {0, 0, 0, 0}, w[8], scale = 0;
                        if (at >= 0) {
                            scale = row_scales<kD>(is_v ? a.vs : a.ks, at);
                            const uint32_t *src = reinterpret_cast<const uint32_t *>(data + at * RB + half * (RB / kHalves)) + p * kWords;
#pragma unroll
                            for (int x = 0; x < kWords; ++x) {
                                c[x] = __ldg(src + x);
                            }
                        }
                        codes16_to_f16<kFmt>(c, w);
                        const uint32_t byte = (scale >> (8 * (half * 2 + (p >> 1)))) & 0xffu;
                        // keys with a block out of range: relative to their largest scale
                        const bool relative = !is_v && !scales_in_range<kD, kFmt>(scale);
                        const int e = relative && byte != 255u ? max(static_cast<int>(byte) + 127 - static_cast<int>(largest_scale<kD>(scale)), 0)
                                                               : static_cast<int>(byte);
                        const float f = __uint_as_float(static_cast<uint32_t>(e) << 23);
                        const float exact = e8m0x2_to_f32(byte).x;
#pragma unroll
                        for (int x = 0; x < 8; ++x) {
                            if (is_v) { // one rounding; NaN for a code or scale that is
                                const float2 v = unpack_16x2<false>(w[x]);
                                w[x] = pack_16x2<kBf16>(v.x * exact, v.y * exact);
                            } else {
                                w[x] = mul_16x2<false>(w[x], pack_16x2<false>(f, f));
                            }
                        }
                        const uint32_t to = dst + half * Sh::kHalfBytes + i * 32 * 128;
                        sts128(to + at0, w[0], w[1], w[2], w[3]);
                        sts128(to + at1, w[4], w[5], w[6], w[7]);
                    }
                }
            }
            fence_proxy_async_smem(); // the tensor core reads through the asynchronous proxy
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&full[slot]);
            }
            if (++slot == ring) {
                slot = 0;
                phase ^= 1u;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        // ------------------------------------------------------------ softmax warps: a thread owns a row
        const int t = warp >> 2, quarter = warp & 3;
        const int row_in_tile = quarter * 32 + lane;
        const int row = (kPair ? 2 * rb + t : rb) * kTile + row_in_tile;
        const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
        const uint32_t s_addr = lane_addr + t * 128, o_addr = lane_addr + 256 + t * 128;
        const uint32_t p_base = smem_u32(smem_p) + t * Sh::kPBytes;
        bool ok = true;
        float row_scale = a.scale_log2 < 0.0f ? -a.scale_log2 : (a.scale_log2 == 0.0f ? 1.0f : a.scale_log2);

        // ---- this row of Q, its sign that of the scale, so that the maximum of the raw logits is that of the scaled
        const int q_tile = kPair ? t : 0;
        if (kPair || t == 0) {
            const uint32_t q_base = smem_u32(smem_q) + q_tile * Sh::kTileBytes;
            const bool live = row < rows;
            const uint16_t *src = nullptr;
            if (live) {
                const int span = a.tokens * a.group;
                const int b = row / span, in = row % span;
                src = a.q + b * a.q_batch + (in / a.group) * a.q_token + static_cast<int64_t>(h * a.group + in % a.group) * a.q_head;
            }
            const uint32_t sign = a.scale_log2 < 0.0f ? 0x80008000u : 0u;
            const uint32_t keep = live && a.scale_log2 != 0.0f ? 0xffffffffu : 0u;
            uint32_t w[kD / 2];
#pragma unroll
            for (int c = 0; c < kD / 8; ++c) {
                const uint4 v = live ? __ldg(reinterpret_cast<const uint4 *>(src) + c) : make_uint4(0, 0, 0, 0);
                w[4 * c] = v.x, w[4 * c + 1] = v.y, w[4 * c + 2] = v.z, w[4 * c + 3] = v.w;
            }
            float factor = 1.0f, inv = 1.0f;
            if constexpr (kBf16 && kMx) {
                uint32_t top = 0; // the largest magnitudes of both halves: bfloat16 pairs order like integers
#pragma unroll
                for (int i = 0; i < kD / 2; ++i) {
                    const uint32_t v = w[i] & 0x7fff7fffu;
                    asm("max.bf16x2 %0, %0, %1;" : "+r"(top) : "r"(v));
                }
                const int field = min(max(static_cast<int>(max(top & 0x7fffu, top >> 16) >> 7), 29), 254);
                factor = __uint_as_float(static_cast<uint32_t>(field - 14) << 23);
                inv = __uint_as_float(static_cast<uint32_t>(254 - (field - 14)) << 23);
            }
#pragma unroll
            for (int c = 0; c < kD / 8; ++c) {
#pragma unroll
                for (int i = 4 * c; i < 4 * c + 4; ++i) {
                    if constexpr (kBf16 && kMx) {
                        const float2 f = unpack_16x2<true>(w[i]);
                        w[i] = pack_16x2<false>(f.x * inv, f.y * inv);
                    }
                    w[i] = (w[i] & keep) ^ sign;
                }
                sts128(q_base + (c >> 3) * Sh::kHalfBytes + swz(row_in_tile, c & 7), w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
            }
            if constexpr (!kPair) {
                ctl->q_factor[row_in_tile] = factor;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ctl->q_full[q_tile]);
            }
            row_scale *= factor;
        } else {
            ok = warp_wait(&ctl->q_full[0], 0, abort_flag, lane);
            row_scale *= ctl->q_factor[kPair ? 0 : row_in_tile];
        }

        const bool rows_here = group_rows[t];
        // Probabilities that become float16 beside V of float16's range are taken 2^7 times as large: at most 2^15, the maximum
        // being up to kDefer behind, they keep every bit down to 2^-21 of the largest
        constexpr float kLift = kBf16 ? 0.0f : 7.0f;
        float m_run = -INFINITY; // reference the probabilities are relative to, raw logits
        float l_run = 0.0f;
        int n = 0;
        for (int j = kPair ? 0 : t; j < tiles && ok && rows_here; j += kPair ? 1 : 2, ++n) {
            if (!warp_wait(&ctl->info_full[j % kInfo], (j / kInfo) & 1, abort_flag, lane) || !warp_wait(&ctl->s_full[t], n & 1, abort_flag, lane)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const Info &info = ctl->info[j % kInfo];
            const bool all_valid = (info.valid[0] & info.valid[1] & info.valid[2] & info.valid[3]) == 0xffffffffu;
            uint32_t flags = 0;
            if constexpr (kMx) {
                flags = info.flags[0] | info.flags[1] | info.flags[2] | info.flags[3];
            }
            const bool plain = all_valid && !(flags & 1u);
            // 64 logits from tensor memory; with the keys' factors, and without the keys that do not exist
            uint32_t x[2][32];
            auto read = [&](int half) {
                tmem_ld_32x32(s_addr + half * 64, x[0]);
                tmem_ld_32x32(s_addr + half * 64 + 32, x[1]);
                tmem_ld_wait();
            };
            auto correct = [&](int half) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t valid = info.valid[2 * half + c];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const float factor = flags & 1u ? __uint_as_float(static_cast<uint32_t>(info.factor[half * 64 + c * 32 + i]) << 16) : 1.0f;
                        x[c][i] = (valid >> i) & 1u ? __float_as_uint(__uint_as_float(x[c][i]) * factor) : 0xff800000u;
                    }
                }
            };
            // ---- first pass: the maximum
            float mx = -INFINITY;
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                read(half);
                if (!plain) {
                    correct(half);
                }
                float m8[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    m8[u] = fmaxf(__uint_as_float(x[0][u]), __uint_as_float(x[1][u]));
#pragma unroll
                    for (int i = 8; i < 32; i += 8) {
                        m8[u] = max3(m8[u], __uint_as_float(x[0][i + u]), __uint_as_float(x[1][i + u]));
                    }
                }
                mx = fmaxf(mx, max3(max3(m8[0], m8[1], m8[2]), max3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7])));
            }
            const float m_new = fmaxf(m_run, mx);
            // also true on the first tile that has a key; false (NaN) while there is none
            const bool grow = (m_new - m_run) * row_scale > kDefer;
            bool pv_waited = n == 0;
            if (__any_sync(0xffffffffu, grow)) {
                if (n > 0) {
                    if (!warp_wait(&ctl->pv_done[t], (n - 1) & 1, abort_flag, lane)) {
                        ok = false;
                        break;
                    }
                    pv_waited = true;
                    tc_fence_after();
                    // rows without a key yet keep their zeros; the others move to the new reference
                    const float alpha = m_run == m_new ? 1.0f : ex2w((m_run - m_new) * row_scale);
                    l_run *= alpha;
#pragma unroll 1
                    for (int d = 0; d < kD / 32; ++d) {
                        uint32_t orow[32];
                        tmem_ld_32x32(o_addr + d * 32, orow);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            orow[i] = __float_as_uint(__uint_as_float(orow[i]) * alpha);
                        }
                        tmem_st_32x32(o_addr + d * 32, orow);
                    }
                    tmem_st_wait();
                    tc_fence_before();
                }
                m_run = m_new;
            }
            // ---- second pass: the probabilities
            const float neg_m = m_run == -INFINITY ? kLift : kBf16 ? -m_run * row_scale : fmaf(-m_run, row_scale, kLift);
            float sum4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {
                read(half);
                if (half == 1) {
                    tc_fence_before();
                    if (lane == 0) {
                        mbar_arrive(&ctl->s_free[t]); // the next S may overwrite this one
                    }
                }
                if (!plain) {
                    correct(half);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float p0 = ex2w(fmaf(__uint_as_float(x[c][i]), row_scale, neg_m));
                        const float p1 = ex2w(fmaf(__uint_as_float(x[c][i + 1]), row_scale, neg_m));
                        sum4[(i >> 1) & 3] += p0 + p1;
                        x[c][i] = __float_as_uint(p0);
                        x[c][i + 1] = __float_as_uint(p1);
                    }
                    // packed in place
                    if (kMx && kBf16 && (flags & 2u)) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            x[c][i] = pack_16x2<true>(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1]));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            x[c][i] = pack_16x2<kOpBf16>(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1]));
                        }
                    }
                    if (c == 0 && !pv_waited) { // the previous product must have read P's buffer
                        ok = warp_wait(&ctl->pv_done[t], (n - 1) & 1, abort_flag, lane);
                        pv_waited = true;
                    }
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        sts128(p_base + half * Sh::kHalfBytes + swz(row_in_tile, c * 4 + q), x[c][4 * q], x[c][4 * q + 1], x[c][4 * q + 2],
                               x[c][4 * q + 3]);
                    }
                }
            }
            if (!ok) {
                break;
            }
            l_run += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&ctl->p_full[t]);
            }
        }
        // ---- (O, m, l) of this group's keys
        if (ok && rows_here) {
            if (n > 0) {
                ok = warp_wait(&ctl->pv_done[t], (n - 1) & 1, abort_flag, lane);
                tc_fence_after();
            }
            const int piece = kPair ? split : 2 * split + t;
            const int64_t slot = (static_cast<int64_t>(piece) * a.kv_heads + h) * a.prefix_tiles + row / kPieceRows;
            const int64_t at = slot * kPieceRows + row % kPieceRows;
            if (ok) {
                if (row < rows) {
                    // without a finite maximum the reference was 0; no key at all: -infinity and no sum
                    a.part_ml[at] = make_float2(m_run != -INFINITY ? (kBf16 ? m_run * row_scale : fmaf(m_run, row_scale, -kLift)) : (l_run == 0.0f ? -INFINITY : -kLift), l_run);
                }
#pragma unroll 1
                for (int c = 0; c < kD / 32 && n > 0; ++c) {
                    uint32_t orow[32];
                    tmem_ld_32x32(o_addr + c * 32, orow);
                    tmem_ld_wait();
                    if (row < rows) {
                        uint4 *dst = reinterpret_cast<uint4 *>(a.part_o + at * kD + c * 32);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            dst[i] = make_uint4(orow[4 * i], orow[4 * i + 1], orow[4 * i + 2], orow[4 * i + 3]);
                        }
                    }
                }
            }
        }
    }

    // ---------------------------------------------------------------- teardown
    tc_fence_before();
    __syncthreads();
    if (ctl->abort_flag) {
        for (int i = 0; i < 1024; ++i) {
            __nanosleep(1000); // products and copies in flight end before shared and tensor memory are given back
        }
        if (threadIdx.x == 0 && atomicCAS(&status->code, 0, kErrDeviceWaitTimeout) == 0) {
            status->block = blockIdx.x;
            status->where = 5;
        }
        __syncthreads();
    }
    if (warp == kIssueWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

template <bool kBf16, int kD, int kFmt, bool kPair>
int launch_one(const AttnArgs &a, DeviceStatus *status, cudaStream_t stream)
{
    using Sh = Shape<kD, kPair>;
    const void *kernel = reinterpret_cast<const void *>(&prefix_wide_kernel<kBf16, kD, kFmt, kPair>);
    // registers move between the warps inside what the block was launched with: with fewer the increase would wait forever
    static const int regs = [kernel] {
        cudaFuncAttributes attr;
        return cudaFuncGetAttributes(&attr, kernel) == cudaSuccess ? attr.numRegs : 0;
    }();
    if (regs != kRegsLaunch) {
        set_error_text("prefix_attn: the kernel was built with %d registers a thread, not %d", regs, kRegsLaunch);
        return kErrUnsupportedShape;
    }
    const int rc = ensure_dynamic_smem(kernel, Sh::kSmem);
    if (rc != kOk) {
        return rc;
    }
    const int rows = a.batch * a.tokens * a.group;
    const int row_blocks = (rows + kTile * Sh::kQTiles - 1) / (kTile * Sh::kQTiles);
    const int64_t blocks = static_cast<int64_t>(a.prefix_splits) * a.kv_heads * row_blocks;
    prefix_wide_kernel<kBf16, kD, kFmt, kPair><<<static_cast<unsigned>(blocks), kThreads, Sh::kSmem, stream>>>(a, status);
    return check_launch();
}

template <bool kBf16, int kD, int kFmt>
int launch_pair(const AttnArgs &a, DeviceStatus *status, cudaStream_t stream)
{
    return a.batch * a.tokens * a.group > kTile ? launch_one<kBf16, kD, kFmt, true>(a, status, stream)
                                                : launch_one<kBf16, kD, kFmt, false>(a, status, stream);
}

template <bool kBf16, int kD>
int launch_fmt(int fmt, const AttnArgs &a, DeviceStatus *status, cudaStream_t stream)
{
    return fmt == kKvMxFp8   ? launch_pair<kBf16, kD, kKvMxFp8>(a, status, stream)
           : fmt == kKvMxFp4 ? launch_pair<kBf16, kD, kKvMxFp4>(a, status, stream)
                             : launch_pair<kBf16, kD, kBf16 ? kKvBf16 : kKvF16>(a, status, stream);
}

} // namespace

int launch_prefix_wide(const AttnArgs &a, int fmt, int d, bool bf16, DeviceStatus *status, cudaStream_t stream)
{
    if (d == 128) {
        return bf16 ? launch_fmt<true, 128>(fmt, a, status, stream) : launch_fmt<false, 128>(fmt, a, status, stream);
    }
    return bf16 ? launch_fmt<true, 64>(fmt, a, status, stream) : launch_fmt<false, 64>(fmt, a, status, stream);
}

} // namespace pto_b200
