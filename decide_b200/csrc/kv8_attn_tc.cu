// dc_kv8_attention for many rows a sequence: the mathematics of kv8_attn.cu on tcgen05.
//
// Products bound it: 4 hd operations for each (pair, key), a pair being a (query row, head of the group), against one exponential
// and one weight to round. A CTA takes 256 pairs that share a kv head as two tiles of 128, the lanes of tensor memory, which pass the
// tensor cores back and forth: while one tile's scores are turned into weights, the other's products run.
//   warps 9..11    codes -> fp16 K and V tiles of 128 keys in shared memory, two stages each. Both lie as rows of keys, 64 columns (128 bytes)
//                 to a swizzled block: K is read as the K-major operand of S = Q K^T, V as the MN-major operand of O += P V, so V needs
//                 no transposition. The 256 pairs share this work.
//   warp 8        issues S = Q K^T and O += P V of the two tiles in turn, 64 keys at a time. A tile has two buffers of scores:
//                 while one is turned into weights the other fills, so that neither side waits for the other's round trip (with one
//                 buffer of 128 keys a step took 4,400 cycles, 1,750 of them between the last weight and the next scores)
//   warps 0..3, 4..7  softmax of a tile, one thread per pair: 64 scores into registers, their maximum, then the weights, which go back
//                 into the columns that the scores came from as the A operand of the V product. Page scales are applied per 16 keys, to
//                 the maximum of a group and inside the exponential's argument: no instruction per score.
// Warp 8 shares its scheduler with two softmax warps and nothing else: with a filler there too its issue of products was the bound.
// The running maximum is lazy as in kv8_attn.cu: O in tensor memory is rescaled only when it grows by more than 2^8.
// Tensor memory: 2 x (2 x 64 columns of scores + 128 of O). Shared memory: q 64 KB, K and V 64 KB each: one CTA an SM. Heads of 256 fill
// both with one tile of 128 pairs (O has 256 columns) and stages of 64 keys; warps 5..7 then help the fillers, who have twice the codes for
// each product (with three of them a half took 3,500 cycles).
// Where there are fewer tiles than SMs the keys are cut into chunks, whose results a second kernel joins in chunk order.
// Measured on the device, 32 query heads of 128 over 8 kv heads: 2,048 rows over 8,191 keys 290 us (829 TFLOP/s), 178 rows over 2,491 keys
// 29 us; kv8_attn.cu takes 1,062 and 51. A round of both tiles' 64 keys takes about 2,000 cycles, its MMAs alone 1,250 (128x64x16 with both
// operands in shared memory 48 each, 128x128x16 with A in tensor memory 64). What it is short of: without the softmax the same call took
// 241 us where the whole took 288 (one warp's issue of products; two warps 185), without its exponentials 266, without the fillers' work 259. Built and measured, and
// slower for it: a warp of products for each tile and six fillers, 512 threads (301 us: the softmax of both tiles then runs in step and
// shares the exponential units); the same with the tiles' exponentials in strict turns (308); scores of 128 keys in one product, which leaves
// room for one buffer a tile (317, though the products alone take 198); fillers in a short loop of single groups (299 to 336); fillers
// whose places are known to the compiler (543: the roles' code no longer fits the instruction cache).
// Every wait is bounded; when one gives up the CTA raises the status word, runs through its steps without waiting, stores nothing, waits for its
// products in flight and returns.
#include "kv8_attn.cuh"
#include "ptx.cuh"

namespace {

using namespace dc;

constexpr uint32_t kHalf = 64;       // keys a product of scores covers
constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;      // S of tile X, buffer B in columns 128 X + 64 B .., O in 256 + 128 X ..
constexpr int kScaleSlots = 4;

template <int HD_>
struct Shape {
    static constexpr int HD = HD_;
    static constexpr int kTiles = 256 / HD;              // tiles of 128 pairs
    static constexpr int kPairs = 128 * kTiles;
    static constexpr int kLd = HD + 4;                   // floats of a pair's partial result
    static constexpr int kHalves = kTiles;               // halves a stage of K or V holds
    static constexpr uint32_t kKeys = kHalf * kHalves;   // keys of a stage
    static constexpr int kGroups = kKeys / 16;           // groups of 16 keys
    // A filler's instruction takes a unit: 512 codes, kRows keys. The 32 units of a stage are shared out evenly, at most kUnits to one.
    static constexpr uint32_t kRows = 512 / HD;
    static constexpr int kFillers = HD == 128 ? 3 : 6;
    static constexpr int kUnits = (32 + kFillers - 1) / kFillers;
    static constexpr uint32_t kQAtom = 128 * 128;        // [128 pairs][64 x 16 bit]
    static constexpr uint32_t kAtom = kKeys * 128;       // [keys][64 x 16 bit]
    static constexpr uint32_t kStage = kAtom * (HD / 64);
    static constexpr uint32_t kQ = 0;                    // [tiles][HD / 64]
    static constexpr uint32_t kK = kQ + kTiles * (HD / 64) * kQAtom;   // [2 stages][HD / 64]
    static constexpr uint32_t kV = kK + 2 * kStage;
    static constexpr uint32_t kScales = kV + 2 * kStage; // float4 [kScaleSlots][8], of 16 keys: K scale hd^-1/2 log2(e), log2 of the V scale, 1 / V scale
    static constexpr uint32_t kRank = kScales + kScaleSlots * 8 * 16;   // float [kPairs]
    static constexpr uint32_t kSeen = kRank + kPairs * 4;   // u32 [kPairs]
    static constexpr uint32_t kBars = kSeen + kPairs * 4;
    static constexpr uint32_t kBytes = kBars + 32 * 8;
};

__device__ __forceinline__ void sts16(uint32_t to, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// A bounded wait that gives no answer: whoever called it goes on as if the phase were complete. A lane that left its loop where the others found the
// phase complete would never meet them again at the next instruction of the whole warp; and for all lanes to agree first takes a vote, 28
// cycles of every wait (2,048 rows over 8,191 keys: 313 us, 292 without). Once one wait has run out the others give up at once, what is worked on is
// in bounds whatever it holds, and nothing is stored.
__device__ __forceinline__ void await(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, int* status, int code) {
    if (mbar_try_wait(bar, parity)) return;
    const uint64_t t0 = globaltimer_ns();
    uint32_t spins = 0;
    while (!mbar_try_wait(bar, parity)) {
        if (*abort_flag) return;
        if ((++spins & 63u) == 0u && globaltimer_ns() - t0 > kWaitLimitNs) {
            *abort_flag = 1u;
            kv8_flag(status, code);
            return;
        }
    }
}

// Advances a two-stage ring.
struct Ring {
    uint32_t stage = 0, phase = 0;
    __device__ __forceinline__ void next() {
        stage ^= 1u;
        if (stage == 0) phase ^= 1u;
    }
};

// V's descriptor: MN-major, 128-byte swizzle. Keys are rows of 128 bytes in groups of 8 (1024 bytes); 64 columns of hd and the next lie `atom` bytes apart.
__device__ __forceinline__ uint64_t desc_mn128(uint32_t smem_addr, uint32_t atom) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
    d |= static_cast<uint64_t>(atom >> 4) << 16;   // leading byte offset: from 64 columns to the next 64
    d |= static_cast<uint64_t>(1024 >> 4) << 32;          // stride byte offset: from 8 keys to the next 8
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}

// Two fp32 operations an instruction: 302 -> 288 us for 2,048 rows over 8,191 keys.
__device__ __forceinline__ uint64_t side_by_side(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 apart(uint64_t x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ uint64_t fma_two(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_two(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 64 keys of a warp's 32 pairs: scores out of tensor memory, their maximum, then the weights into the columns that the scores came from.
// MASKED: some pair of the warp does not see all 64 keys; `vis` of them it does. settled(): O may be rescaled.
template <int HD, bool MASKED, typename F>
__device__ __forceinline__ void softmax_half(uint32_t col_s, uint32_t col_o, const float4* sc, float mul, int vis, bool scale_o, float& m, float& l, F settled) {
    uint32_t s[2][32];
    tmem_ld_32x32(col_s, s[0]);
    tmem_ld_32x32(col_s + 32, s[1]);
    tmem_ld_wait();
    float top = kKv8None;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        uint32_t* v = s[g >> 1] + 16 * (g & 1);
        float t[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
            if (MASKED) {
                v[e] = 16 * g + e < vis ? v[e] : 0xff800000u;   // out of the maximum
                v[e + 1] = 16 * g + e + 1 < vis ? v[e + 1] : 0xff800000u;
            }
            t[(e >> 1) & 1] = fmaxf(fmaxf(t[(e >> 1) & 1], __uint_as_float(v[e])), __uint_as_float(v[e + 1]));
        }
        const float2 ab = *reinterpret_cast<const float2*>(sc + g);
        top = fmaxf(top, fmaf(fmaxf(t[0], t[1]), mul * ab.x, ab.y));
    }
    const bool grow = top > m + kKv8Step;
    if (__any_sync(0xffffffffu, grow)) {
        // O and the total follow the new maximum (pairs whose maximum stays put scale by 1)
        const float to = grow ? top - kKv8Below : m, by = ex2(m - to);
        l *= by;
        m = to;
        if (scale_o) {
            settled();
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
                uint32_t v[16];
                tmem_ld_32x32_x16(col_o + 16 * c, v);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = __float_as_uint(__uint_as_float(v[e]) * by);
                tmem_st_32x32_x16(col_o + 16 * c, v);
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t w[16];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const uint32_t* v = s[h] + 16 * g;
            const float4 ab = sc[2 * h + g];
            const uint64_t by = side_by_side(mul * ab.x, mul * ab.x), off = side_by_side(ab.y - m, ab.y - m);
            uint64_t sums = side_by_side(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
                const float2 t = apart(fma_two(side_by_side(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), by, off));
                float p0 = ex2(t.x), p1 = ex2(t.y);
                if (MASKED) {   // explicitly: a scale that is NaN, or a multiplier of zero, makes no zero of -infinity
                    p0 = 32 * h + 16 * g + e < vis ? p0 : 0.f;
                    p1 = 32 * h + 16 * g + e + 1 < vis ? p1 : 0.f;
                }
                // cut to fp16's 11 bits, then exact in fp16 from 2^-14 on: product and total take the same weight, and what the cut does to all
                // of a row's weights alike cancels: error against 64 bits 1.2 instead of 1.3 times that of rounding the output, for 10 of 290 us of
                // 2,048 rows over 8,191 keys (of weights rounded to nearest, as kv8_attn.cu has them, the total cost three instructions each, 57 us)
                p0 = __uint_as_float(__float_as_uint(p0) & 0xffffe000u);
                p1 = __uint_as_float(__float_as_uint(p1) & 0xffffe000u);
                w[8 * g + e / 2] = ActF16::pack(p0, p1);
                sums = add_two(sums, side_by_side(p0, p1));
            }
            const float2 sum = apart(sums);
            l = fmaf(sum.x + sum.y, ab.z, l);
        }
        tmem_st_32x32_x16(col_s + 16 * h, w);
    }
}

template <typename Act, int HD>
__global__ void __launch_bounds__(kThreads, 1) kv8_attn_tc_kernel(const Kv8Args a) {
    using S = Shape<HD>;
    constexpr int kPairs = S::kPairs, kLd = S::kLd;
    constexpr uint32_t kKeys = S::kKeys;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint64_t* k_full = bars;            // [2] the fillers have written K
    uint64_t* v_full = bars + 2;        // [2]
    uint64_t* k_free = bars + 4;        // [2] both tiles' score products are done
    uint64_t* v_free = bars + 6;        // [2]
    uint64_t* s_full = bars + 8;        // [2 tiles][2 buffers] scores are there
    uint64_t* p_full = bars + 12;       // [2][2] the tile's four warps have written the weights (and rescaled O)
    uint64_t* pv_done = bars + 16;      // [2] a V product of the tile, and every product before it, is done
    uint64_t* scale_full = bars + 18;   // [kScaleSlots]
    uint64_t* q_full = bars + 22;       // warps 0..7 have written q
    uint64_t* drain_bar = bars + 23;
    uint64_t* o_full = bars + 24;       // [2] the tile's last product is done
    uint64_t* l_full = bars + 26;       // heads of 256: the pairs' divisors are there
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 27);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    volatile uint32_t* never_flag = tmem_slot + 2;
    float4* scales = reinterpret_cast<float4*>(smem + S::kScales);
    float* rank = reinterpret_cast<float*>(smem + S::kRank);
    uint32_t* seen = reinterpret_cast<uint32_t*>(smem + S::kSeen);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    kv8_begin();
    uint32_t id = blockIdx.x;
    const uint32_t z = id % a.chunks;
    id /= a.chunks;
    const uint32_t tile_id = id, kvh = id % a.c.nkv;
    id /= a.c.nkv;
    const uint32_t mt = a.tiles - 1 - id % a.tiles, j = id / a.tiles;   // the last rows, which see the most keys, first

    const Kv8Rows r = kv8_rows(a.c, a.q_start, j, a.rows, a.max_q);
    const bool reports = kvh == 0 && z == 0;
    if (!r.ok) {
        if (reports && tid == 0) kv8_flag(a.status, DC_STATUS_KV8_OFFSETS);
        return;
    }
    const uint32_t pair0 = mt * kPairs, pairs = r.count * a.group;
    if (pair0 >= pairs) return;
    if (r.len > a.max_len) {
        if (reports && tid == 0) kv8_flag(a.status, DC_STATUS_KV8_LENGTH);
        return;
    }
    const uint32_t here = min(static_cast<uint32_t>(kPairs), pairs - pair0);
    const bool two = S::kTiles == 2 && here > 128;   // the second tile has rows

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], S::kFillers);
            mbar_init(&v_full[i], S::kFillers);
            mbar_init(&k_free[i], 1);
            mbar_init(&v_free[i], 1);
            mbar_init(&pv_done[i], 1);
            mbar_init(&o_full[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        for (int i = 0; i < kScaleSlots; ++i) mbar_init(&scale_full[i], 1);
        mbar_init(q_full, two ? 8 : 4);
        mbar_init(drain_bar, 1);
        mbar_init(l_full, 4);
        *abort_flag = 0u;
        *never_flag = 0u;
        fence_mbar_init();
    }
    if (warp == 8) {
        tmem_alloc(tmem_slot, kTmemCols);
        tmem_relinquish();
    }
    // tokens that the pairs attend, and the most that any of them does: every warp for itself, so that none waits for another
    uint32_t most = 0;
    {
        bool past = false;
#pragma unroll
        for (int i = 0; i < kPairs / 32; ++i) {
            const uint32_t p = 32 * i + lane, n = p < here ? kv8_visible(r, a.qpos, kv8_row_of(a, pair0 + p), &past) : 0u;
            if (warp == i) seen[p] = n;
            most = max(most, n);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        if (past && reports && warp == 0) kv8_flag(a.status, DC_STATUS_KV8_POSITION);
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t key0 = z * a.chunk;
    const bool whole = most <= a.chunk;
    const bool idle = z && key0 >= most;             // nothing of this tile in this chunk
    const uint32_t key1 = min(most, key0 + a.chunk);
    const uint32_t halves = idle ? 0u : (key1 - key0 + kHalf - 1) / kHalf, steps = (halves + S::kHalves - 1) / S::kHalves;
    const uint32_t tmem = *tmem_slot;                // 0: all of it is ours

    float m = kKv8None, l = 0.f;                     // softmax warps: of their pair
    if (warp > 8 || (HD == 256 && warp > 4 && warp < 8)) {
        // -------------------------------------------------------------------------------- codes -> fp16 tiles
        constexpr int kUnits = S::kUnits;
        constexpr uint32_t kRows = S::kRows, kPerGroup = 16 / kRows;   // keys of a unit, units of a group of 16 keys
        const int w = HD == 128 || warp < 8 ? (HD == 128 ? warp - 9 : warp - 5) : warp - 6, unit0 = 32 * w / S::kFillers, units = 32 * (w + 1) / S::kFillers - unit0;
        const uint32_t token = static_cast<uint32_t>(a.c.token_stride), unit_step = kRows * token;   // strides below 2^28: up to 15 of them fit 32 bits
        const uint32_t* table = a.c.table + static_cast<size_t>(j) * a.c.max_pages;
        // A lane's place in a unit: row bits from lane bits 2 and (of four rows) 4, 16-code piece c from bits 0, 1 and the others, so that the
        // eight lanes of a store's phase, four pieces of two rows, meet all 32 banks of the swizzled tile.
        const uint32_t fr = HD == 128 ? ((lane >> 2) & 1) | ((lane >> 4) << 1) : (lane >> 2) & 1;
        const uint32_t c = HD == 128 ? (lane & 3) | ((lane >> 1) & 4) : (lane & 3) | ((lane >> 3) << 2);
        const uint8_t* kc = static_cast<const uint8_t*>(a.c.k) + kvh * a.c.head_stride + fr * token + 16 * c;
        const int64_t to_v = static_cast<const uint8_t*>(a.c.v) - static_cast<const uint8_t*>(a.c.k);
        // The filler's units lie in up to kGroups groups of 16 keys, whose pages every lane looks up for itself, a step ahead of the codes.
        constexpr int kGroups = HD == 128 ? 4 : 2;
        const uint32_t group0 = unit0 / kPerGroup;
        uint32_t page[kGroups];
        auto look_up = [&](uint32_t step) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const uint32_t key = key0 + step * kKeys + 16 * (group0 + g);
                page[g] = key < key1 && group0 + g < S::kGroups ? __ldg(table + (key >> a.page_shift)) : 0u;
            }
        };
        const uint8_t* at[kGroups];   // first code of the group in K, this lane's; V lies at the same distance from its first
        // What stands in for a page outside the pool has to hold numbers, or pairs that do not attend it would take the code for NaN times a weight of
        // zero: the sequence's first page, which is full where a later one is attended. Where the first is itself outside the pool every
        // pair that attends anything is NaN. (Zeros instead, chosen at each load, took 12 % of the time of 2,048 rows over 8,191 keys.)
        auto to_page = [&](uint32_t step) {
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const uint32_t key = key0 + step * kKeys + 16 * (group0 + g);
                if (page[g] >= a.c.n_pages) {
                    kv8_flag(a.status, DC_STATUS_KV8_PAGE);
                    page[g] = __ldg(table);
                    if (page[g] >= a.c.n_pages) page[g] = 0;
                }
                at[g] = kc + page[g] * a.c.page_stride + (key & (a.c.page_size - 1)) * a.c.token_stride;   // 64 bits: up to 112 strides of 2^28
            }
        };
        uint4 kx[kUnits], vx[kUnits];
        auto load = [&](uint4 (&x)[kUnits], int64_t from, uint32_t step) {   // rows kRows (unit0 + i) + fr; zeros past the last token
            const uint32_t first = key0 + step * kKeys + kRows * unit0 + fr;
            const bool inside = key0 + (step + 1) * kKeys <= key1;
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                if (i >= 32 / S::kFillers && i >= units) break;
                const uint32_t u = unit0 % kPerGroup + i;   // from the start of the first group
                const uint8_t* group = at[0];
#pragma unroll
                for (int g = 1; g < kGroups; ++g) group = u < g * kPerGroup ? group : at[g];
                if (inside || first + kRows * i < key1) x[i] = __ldg(reinterpret_cast<const uint4*>(group + from + (u % kPerGroup) * unit_step));
                else x[i] = make_uint4(0, 0, 0, 0);
            }
        };
        // filler 0 also keeps the scales of the stage's groups, lane g those of group g
        uint32_t scale_page = 0;
        bool scale_there = false;   // the group has a key that some pair attends: others have no page whose scale means anything
        float k_scale = 0.f, v_scale = 1.f;
        auto scale_look_up = [&](uint32_t step) {
            const uint32_t key = key0 + step * kKeys + 16 * (lane % S::kGroups);
            scale_there = key < key1;
            scale_page = scale_there ? __ldg(table + (key >> a.page_shift)) : 0u;
        };
        auto scale_load = [&] {
            const size_t s = static_cast<size_t>(scale_page < a.c.n_pages ? scale_page : 0u) * a.c.nkv + kvh;
            k_scale = a.c.k_scale[s];
            v_scale = a.c.v_scale[s];
            if (scale_page >= a.c.n_pages) k_scale = __uint_as_float(0x7fffffffu);   // what attends it is NaN
            if (!scale_there) k_scale = v_scale = 1.f;
        };
        // 16 codes become the 16-byte pieces 2 c and 2 c + 1 of the row, eight pieces to an atom, at piece ^ (row % 8): with row = kRows u + fr that
        // is one address and its neighbour at ^ 16, both at ^ 16 (kRows u % 8)
        const uint32_t to0 = smem_u32(smem) + (c >> 2) * S::kAtom + (kRows * unit0 + fr) * 128 + (((2 * c) ^ fr) & 7) * 16;
        auto store = [&](const uint4 (&x)[kUnits], uint32_t tile) {
            const uint32_t to = to0 + tile;
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                if (i >= 32 / S::kFillers && i >= units) break;
                const uint32_t swizzle = 16 * (kRows * (unit0 + i) & 7), at_unit = (to ^ swizzle) + kRows * 128 * i, beside = (to ^ swizzle ^ 16) + kRows * 128 * i;
                sts16(at_unit, low_codes(x[i].x), high_codes(x[i].x), low_codes(x[i].y), high_codes(x[i].y));
                sts16(beside, low_codes(x[i].z), high_codes(x[i].z), low_codes(x[i].w), high_codes(x[i].w));
            }
        };
        Ring ring;
        if (steps) {
            look_up(0);
            if (w == 0) scale_look_up(0);
            to_page(0);
            load(kx, 0, 0);
            load(vx, to_v, 0);
            if (w == 0) {
                scale_load();
                scale_look_up(1);
            }
            look_up(1);
        }
        for (uint32_t i = 0; i < steps; ++i) {
            if (i >= 2) await(&k_free[ring.stage], ring.phase ^ 1u, abort_flag, a.status, 81);
            if (w == 0 && lane < S::kGroups) {
                const float e = kv8_log2i(v_scale);   // a NaN reaches the total through the weights, not through 1 / V scale
                scales[(i % kScaleSlots) * 8 + lane] = make_float4(a.scale * k_scale, e, isnan(e) ? 1.f : kv8_exp2i(max(-126, min(127, -static_cast<int>(e)))), 0.f);
            }
            store(kx, S::kK + ring.stage * S::kStage);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (w == 0) mbar_arrive(&scale_full[i % kScaleSlots]);
                mbar_arrive(&k_full[ring.stage]);
            }
            const bool more = i + 1 < steps;
            if (more) {
                to_page(i + 1);
                load(kx, 0, i + 1);
            }
            if (i >= 2) await(&v_free[ring.stage], ring.phase ^ 1u, abort_flag, a.status, 82);
            store(vx, S::kV + ring.stage * S::kStage);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[ring.stage]);
            if (more) {
                load(vx, to_v, i + 1);
                if (w == 0) {
                    scale_load();
                    scale_look_up(i + 2);
                }
                look_up(i + 2);
            }
            ring.next();
        }
    } else if (warp == 8) {
        // -------------------------------------------------------------------------------- products
        // The whole warp walks the steps and one elected lane issues. Operands of an MMA come from uniform registers: four halves are unrolled,
        // so that every address is a constant (shared memory starts at a constant, and who owns all of tensor memory starts at column 0).
        // With addresses worked out at run time an MMA took 60 to 70 cycles to issue, more than it takes to run.
        if (steps) {
            constexpr uint32_t idesc_s = umma_idesc(0, 0, 128, kHalf), idesc_o = umma_idesc(0, 0, 128, HD) | (1u << 16);   // B of the V product is MN-major
            constexpr uint64_t kQStep = S::kQAtom >> 4, kStep = S::kAtom >> 4, kStageStep = S::kStage >> 4, kHalfStep = kHalf * 128 >> 4;   // 64 keys: 64 rows of 128 bytes
            constexpr int kShift = S::kHalves - 1;   // half h lies in stage (h >> kShift) & 1
            const uint64_t dq = umma_desc_k128(smem_u32(smem) + S::kQ), dk = umma_desc_k128(smem_u32(smem) + S::kK), dv = desc_mn128(smem_u32(smem) + S::kV, S::kAtom);
            const uint32_t n = halves;
            const bool both = two;
            auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
                await(bar, parity, abort_flag, a.status, code);
                __syncwarp();
            };
            // half u of a round of four: buffer u % 2; `last`: the stage's last product of the kind
            auto scores = [&](int x, int u, bool last) {
                const int stage = u >> kShift & 1, part = S::kHalves == 2 ? u & 1 : 0;
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ++ks) {
                        const uint64_t da = dq + (x * (HD / 64) + (ks >> 2)) * kQStep + 2 * (ks & 3);
                        const uint64_t db = dk + (stage * kStageStep + part * kHalfStep + (ks >> 2) * kStep + 2 * (ks & 3));
                        if (ks == 0) umma_bf16_ss<false>(128 * x + 64 * (u & 1), da, db, idesc_s);
                        else umma_bf16_ss<true>(128 * x + 64 * (u & 1), da, db, idesc_s);
                    }
                    umma_commit(&s_full[2 * x + (u & 1)]);
                    if (last) umma_commit(&k_free[stage]);
                }
                __syncwarp();
            };
            auto values = [&](int x, int u, bool first, bool last, bool over) {
                const int stage = u >> kShift & 1, part = S::kHalves == 2 ? u & 1 : 0;
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks) {   // 16 keys: 8 columns of weights, 2048 bytes of V
                        const uint64_t db = dv + (stage * kStageStep + part * kHalfStep + ks * (2048 >> 4));
                        if (ks == 0 && first) umma_bf16_ts<false>(kColO + 128 * x, 128 * x + 64 * (u & 1) + 8 * ks, db, idesc_o);
                        else umma_bf16_ts<true>(kColO + 128 * x, 128 * x + 64 * (u & 1) + 8 * ks, db, idesc_o);
                    }
                    umma_commit(&pv_done[x]);
                    if (last) umma_commit(&v_free[stage]);
                    if (over) umma_commit(&o_full[x]);
                }
                __syncwarp();
            };
            constexpr bool kOwn = S::kHalves == 1;   // every half is a stage of its own
            wait(q_full, 0u, 83);
            wait(&k_full[0], 0u, 83);
            tc_fence_after_sync();
            scores(0, 0, kOwn || (!both && n == 1));
            if (both) scores(1, 0, n == 1);
            if (n > 1) {
                if (kOwn) wait(&k_full[1], 0u, 83);
                if (kOwn) tc_fence_after_sync();
                scores(0, 1, !both);
                if (both) scores(1, 1, true);
            }
            // A wait costs some 150 cycles even when it is over: each stands right behind products that were just issued.
            for (uint32_t h0 = 0; h0 < n; h0 += 4) {
                const uint32_t phase = h0 >> 2 & 1;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint32_t h = h0 + u;
                    if (h >= n) break;
                    wait(&p_full[u & 1], u >> 1, 84);
                    if (kOwn || !(u & 1)) wait(&v_full[u >> kShift & 1], kOwn ? u >> 1 : phase, 85);
                    tc_fence_after_sync();
                    const bool more = h + 2 < n, ends = kOwn || (u & 1) || h + 1 == n, next_ends = kOwn || (u & 1) || h + 3 == n;
                    values(0, u, u == 0 && h0 == 0, !both && ends, h + 1 == n);
                    if (both) wait(&p_full[2 + (u & 1)], u >> 1, 84);
                    if (more && (kOwn || !(u & 1))) wait(&k_full[(u + 2) >> kShift & 1], kOwn ? (u >> 1) ^ 1 : (u ? phase ^ 1u : phase), 86);
                    tc_fence_after_sync();
                    if (more) scores(0, u + 2, !both && next_ends);
                    if (both) {
                        values(1, u, u == 0 && h0 == 0, ends, h + 1 == n);
                        if (more) scores(1, u + 2, next_ends);
                    }
                }
            }
        }
    } else {
        // -------------------------------------------------------------------------------- softmax: one thread per pair
        const uint32_t x = warp >> 2, p = tid;       // tile; pair of the CTA
        const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16), col_o = lanes + kColO + 128 * x;
        const bool runs = x == 0 || two;
        if (runs && halves) {
            // q of the warp's 32 pairs: 16 bytes a lane, eight instructions' rows on their way together; bf16 rows are brought into
            // fp16's range as in kv8_attn.cu. The loops here and at the end are rolled: code that runs once costs its way from memory.
            constexpr uint32_t kLanes = HD / 8, kAtOnce = 32 / kLanes;   // lanes of a row, rows of an instruction
            const uint32_t piece = lane % kLanes;
            uint8_t* to = smem + S::kQ + (x * (HD / 64) + (piece >> 3)) * S::kQAtom;
#pragma unroll 1
            for (uint32_t p0 = 32 * warp + lane / kLanes; p0 < 32 * warp + 32; p0 += 8 * kAtOnce) {
                uint4 v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t pair = pair0 + p0 + kAtOnce * i, of = kv8_row_of(a, pair), h = kvh * a.group + pair - of * a.group;
                    v[i] = p0 + kAtOnce * i < here ? *reinterpret_cast<const uint4*>(a.q + static_cast<size_t>(r.start + of) * a.ldq + static_cast<size_t>(h) * HD + 8 * piece) : make_uint4(0, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t row = (p0 + kAtOnce * i) & 127;
                    uint2 w[2] = {make_uint2(v[i].x, v[i].y), make_uint2(v[i].z, v[i].w)};
                    const float up = kv8_query_row<Act, 2>(w, kv8_query_top<2>(w, kLanes));
                    if (piece == 0) rank[p0 + kAtOnce * i] = up;
                    // 16-byte piece of the row, swizzled by the row
                    *reinterpret_cast<uint4*>(to + row * 128 + (((piece & 7) ^ (row & 7)) << 4)) = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        }
        const bool on = p < here;
        const float mul = runs && halves ? rank[p] : 0.f;
        const uint32_t see = on ? seen[p] : most;    // pairs past the last are computed (their q is zero) and not stored
        for (uint32_t h = 0; runs && h < halves; ++h) {
            const uint32_t step = h / S::kHalves;
            await(&scale_full[step % kScaleSlots], step / kScaleSlots & 1u, abort_flag, a.status, 88);
            await(&s_full[2 * x + (h & 1)], h >> 1 & 1, abort_flag, a.status, 89);
            __syncwarp();
            tc_fence_after_sync();
            const float4* sc = scales + step % kScaleSlots * 8 + 4 * (h % S::kHalves);
            const uint32_t key = key0 + h * kHalf, col_s = lanes + 128 * x + 64 * (h & 1);
            const int vis = static_cast<int>(min(see, key + kHalf)) - static_cast<int>(min(see, key));   // of the 64 keys
            auto settled = [&] {   // the V product of the last 64 keys: the one before it came before these scores, the next has no weights yet
                await(&pv_done[x], (h - 1) & 1u, abort_flag, a.status, 91);
                __syncwarp();
                tc_fence_after_sync();
            };
            if (__any_sync(0xffffffffu, vis < static_cast<int>(kHalf))) softmax_half<HD, true>(col_s, col_o, sc, mul, vis, h > 0, m, l, settled);
            else softmax_half<HD, false>(col_s, col_o, sc, mul, vis, h > 0, m, l, settled);
            tmem_st_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * x + (h & 1)]);
        }
        // the divisor, for whoever stores the pair's columns
        if (HD == 256 && x == 0 && !idle) {
            rank[p] = l == 0.f ? 0.f : whole ? 1.0f / l : 1.0f;
            __syncwarp();
            if (lane == 0) mbar_arrive(l_full);
        }
    }

    // ------------------------------------------------------------------------------------ output
    // Warps 0..7, 32 pairs each; of heads of 256, warps 0..3 store columns 0..127 of the tile's pairs and warps 4..7 the others (a warp reaches the
    // lanes of tensor memory that its number modulo four gives). A tile's q is free once its last product is done (its scores came
    // before it): rows go through 8 KB of it, 64 columns at a time, so that they leave in whole pieces. Row r keeps its 16-byte pieces at
    // piece ^ (r % 16).
    if (warp < 8 && !idle && (HD == 256 || warp < 4 || two)) {
        const uint32_t x = HD == 256 ? 0 : warp >> 2, part = HD == 256 ? warp >> 2 : 0, first = HD == 256 ? 32 * (warp & 3) : 32 * warp;   // tile, 128 columns, pair of lane 0
        // (pv_done cannot tell: it may have run two phases ahead, and a wait for a phase that lies two back waits for the next one like it)
        if (HD == 256) await(l_full, 0u, abort_flag, a.status, 92);
        if (halves) await(&o_full[x], 0u, abort_flag, a.status, 90);
        __syncwarp();
        tc_fence_after_sync();
        if (__all_sync(0xffffffffu, *abort_flag == 0u)) {
            uint8_t* stage = smem + S::kQ + warp * 8192;
            const float by = HD == 256 ? rank[first + lane] : l == 0.f ? 0.f : whole ? 1.0f / l : 1.0f;   // 0: the pair attends nothing here, whatever lies in O
            const uint32_t col8 = lane & 7, col_o = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16) + kColO + 128 * (x + part);   // eight lanes a row
            float* parts = a.part + (static_cast<size_t>(tile_id) * a.chunks + z) * kPairs * kLd;
            if (!whole && part == 0 && first + lane < here) *reinterpret_cast<float2*>(parts + (first + lane) * kLd + HD) = make_float2(m, l);
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
                const uint32_t d = 128 * part + 64 * c;
                // the gates of the eight rows that this lane will store are asked for first (asked for row by row they took 24 us of a tile)
                float4 gate[8][2];
                if (whole && a.gate) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t pr = first + 4 * i + (lane >> 3);
                        if (pr < here) kv8_gate8(a, r, pair0 + pr, kvh, d + 8 * col8, HD, gate[i]);
                    }
                }
                __syncwarp();
#pragma unroll 1
                for (int q4 = 0; q4 < 4; ++q4) {
                    uint32_t v[16];
                    if (halves) {
                        tmem_ld_32x32_x16(col_o + 64 * c + 16 * q4, v);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        uint4 o = make_uint4(0, 0, 0, 0);
                        if (halves && by != 0.f) o = make_uint4(__float_as_uint(__uint_as_float(v[e]) * by), __float_as_uint(__uint_as_float(v[e + 1]) * by),
                                                   __float_as_uint(__uint_as_float(v[e + 2]) * by), __float_as_uint(__uint_as_float(v[e + 3]) * by));
                        *reinterpret_cast<uint4*>(stage + lane * 256 + (((4 * q4 + e / 4) ^ (lane & 15)) << 4)) = o;
                    }
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; ++i) {                       // four rows at a time
                    const uint32_t rr = 4 * i + (lane >> 3), pr = first + rr;
                    // 16 bytes of output are 8 columns, side by side; 16 bytes of a partial result are 4: a lane's two pieces lie apart, so
                    // that the lanes of a row fill whole sectors
                    const uint32_t p0 = whole ? 2 * col8 : col8, p1 = whole ? p0 + 1 : p0 + 8;
                    const float4 o0 = *reinterpret_cast<const float4*>(stage + rr * 256 + ((p0 ^ (rr & 15)) << 4));
                    const float4 o1 = *reinterpret_cast<const float4*>(stage + rr * 256 + ((p1 ^ (rr & 15)) << 4));
                    if (pr >= here) continue;
                    if (whole) {
                        kv8_store8<Act>(a, r, pair0 + pr, kvh, d + 8 * col8, HD, o0, o1, gate[i]);
                    } else {
                        *reinterpret_cast<float4*>(parts + pr * kLd + d + 4 * p0) = o0;
                        *reinterpret_cast<float4*>(parts + pr * kLd + d + 4 * p1) = o1;
                    }
                }
            }
        }
    }

    // ------------------------------------------------------------------------------------ teardown
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 8) {
        if (*abort_flag) {   // no product may still be writing tensor memory when it is freed
            if (elect_one()) umma_commit(drain_bar);
            __syncwarp();
            mbar_wait(drain_bar, 0u, never_flag, a.status, 87);
        }
        tc_fence_after_sync();
        __syncwarp();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Joins the chunks of some pairs of a tile, in chunk order; a thread takes 8 columns of a pair. Tiles that one chunk held are done already.
template <typename Act, int HD>
__global__ void __launch_bounds__(256) kv8_join_kernel(const Kv8Args a) {
    constexpr int kPairs = Shape<HD>::kPairs, kLd = Shape<HD>::kLd, kCols = HD / 8, kHere = 256 / kCols;   // threads of a pair, pairs of a CTA
    kv8_begin();
    const uint32_t tile_id = blockIdx.x / (kPairs / kHere), p = blockIdx.x % (kPairs / kHere) * kHere + threadIdx.x / kCols, d = threadIdx.x % kCols * 8;
    const uint32_t kvh = tile_id % a.c.nkv, mt = a.tiles - 1 - tile_id / a.c.nkv % a.tiles, j = tile_id / a.c.nkv / a.tiles;
    const Kv8Rows r = kv8_rows(a.c, a.q_start, j, a.rows, a.max_q);
    if (!r.ok || r.len > a.max_len) return;
    const uint32_t pair0 = mt * kPairs, pairs = r.count * a.group;
    if (pair0 >= pairs) return;
    const uint32_t here = min(static_cast<uint32_t>(kPairs), pairs - pair0);
    __shared__ uint32_t most_at;
    if (threadIdx.x == 0) most_at = 0;
    __syncthreads();
    bool past = false;
    uint32_t n = threadIdx.x < here ? kv8_visible(r, a.qpos, kv8_row_of(a, pair0 + threadIdx.x), &past) : 0u;
    n = __reduce_max_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) atomicMax(&most_at, n);
    __syncthreads();
    const uint32_t most = most_at;
    if (most <= a.chunk || p >= here) return;
    const uint32_t chunks = (most + a.chunk - 1) / a.chunk;
    const float* from = a.part + (static_cast<size_t>(tile_id) * a.chunks * kPairs + p) * kLd;
    constexpr size_t kStepFloats = static_cast<size_t>(kPairs) * kLd;
    float top = kKv8None, total = 0.f, x[8] = {};
    for (uint32_t k = 0; k < chunks; ++k) top = fmaxf(top, from[k * kStepFloats + HD]);
#pragma unroll 4
    for (uint32_t k = 0; k < chunks; ++k) {
        const float* at = from + k * kStepFloats;
        const float2 ml = *reinterpret_cast<const float2*>(at + HD);
        const float4 u = *reinterpret_cast<const float4*>(at + d), w = *reinterpret_cast<const float4*>(at + d + 4);
        const float by = ex2(ml.x - top), v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
        total = fmaf(ml.y, by, total);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fmaf(v[i], by, x[i]);
    }
    kv8_finish<Act>(a, r, pair0 + p, kvh, d, HD, total, x);
}

}  // namespace

int dc_kv8_attention_tc_warm(dc_ctx* ctx) {
    static bool set[16] = {};
    if (set[ctx->device & 15]) return DC_OK;
    typedef void (*fn)(const Kv8Args);
    const fn all[4] = {kv8_attn_tc_kernel<ActF16, 128>, kv8_attn_tc_kernel<ActBF16, 128>, kv8_attn_tc_kernel<ActF16, 256>, kv8_attn_tc_kernel<ActBF16, 256>};
    for (int i = 0; i < 4; ++i) {
        const int bytes = static_cast<int>(i < 2 ? Shape<128>::kBytes : Shape<256>::kBytes);
        const cudaError_t e = cudaFuncSetAttribute(all[i], cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return dc_fail(ctx, DC_CUDA_ERROR, "kv8_attention: cannot opt in to %d bytes of shared memory: %s", bytes, cudaGetErrorString(e));
    }
    set[ctx->device & 15] = true;
    return DC_OK;
}

// How a call is cut: tiles of 256 pairs (heads of 256: 128); where there are fewer of them than SMs, the keys in chunks of at least 256.
Kv8Cut dc_kv8_attention_tc_cut(const dc_ctx* ctx, const dc_kv8_cache* c, uint32_t nq, uint32_t max_q, uint32_t max_len) {
    Kv8Cut t;
    const uint64_t pairs = static_cast<uint64_t>(max_q) * (nq / c->nkv), wide = c->hd == 128 ? Shape<128>::kPairs : Shape<256>::kPairs;
    t.tiles = static_cast<uint32_t>((pairs + wide - 1) / wide);
    const uint64_t whole = static_cast<uint64_t>(c->n_seqs) * c->nkv * t.tiles;
    uint64_t parts = static_cast<uint64_t>(ctx->sm_count) / whole;
    const uint64_t most = (max_len + 255) / 256;
    parts = parts < 1 ? 1 : parts > most ? most : parts;
    t.chunk = static_cast<uint32_t>(((max_len + parts - 1) / parts + 127) / 128 * 128);
    t.chunks = (max_len + t.chunk - 1) / t.chunk;
    t.ctas = whole * t.chunks;
    t.part_bytes = t.chunks > 1 ? t.ctas * wide * (c->hd + 4) * sizeof(float) : 0;
    return t;
}

int dc_kv8_attention_tc(dc_ctx* ctx, cudaStream_t s, const dc::Kv8Args& a, uint64_t ctas) {
    const int rc = dc_kv8_attention_tc_warm(ctx);
    if (rc != DC_OK) return rc;
    const bool f16 = ctx->act_dtype == DC_ACT_F16, narrow = a.c.hd == 128;
    auto kern = narrow ? (f16 ? kv8_attn_tc_kernel<ActF16, 128> : kv8_attn_tc_kernel<ActBF16, 128>) : (f16 ? kv8_attn_tc_kernel<ActF16, 256> : kv8_attn_tc_kernel<ActBF16, 256>);
    const int launched = dc_kv8_launch(ctx, "kv8_attention (tcgen05)", kern, false, dim3(static_cast<uint32_t>(ctas)), kThreads, narrow ? Shape<128>::kBytes : Shape<256>::kBytes, s, a);
    if (launched != DC_OK || a.chunks == 1) return launched;
    auto join = narrow ? (f16 ? kv8_join_kernel<ActF16, 128> : kv8_join_kernel<ActBF16, 128>) : (f16 ? kv8_join_kernel<ActF16, 256> : kv8_join_kernel<ActBF16, 256>);
    const uint32_t per_tile = narrow ? Shape<128>::kPairs / 16 : Shape<256>::kPairs / 8;
    return dc_kv8_launch(ctx, "kv8_attention (join)", join, true, dim3(static_cast<uint32_t>(ctas / a.chunks * per_tile)), 256, 0, s, a);
}
