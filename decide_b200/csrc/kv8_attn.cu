// dc_kv8_attention: causal GQA attention over one layer of the paged 8-bit K/V cache.
//
// The mathematics. With codes k', v' and page scales a = 2^e_k, b = 2^e_v (per page and kv head), row r of head h has scores
// s_j = a_j (q . k'_j) hd^-1/2 and o = sum_j softmax(s)_j b_j v'_j. Taking the V scale into the exponent, with t_j = s_j log2(e) + e_v(j):
//     o = sum_j 2^(t_j - m) v'_j / sum_j 2^(t_j - m) 2^-e_v(j),    m any upper bound of t_j up to a factor,
// so that one running maximum serves both sums, the weights of the V product are relative to the row's largest TERM, and no code is
// ever scaled: codes go into the tensor cores as fp16, exactly. The sum of the weights is fp32, before they are rounded to fp16.
//
// K/V bytes bound it when there are few rows. A tile of up to 16 (query row, head of the group) pairs shares a kv head's codes; the
// warps of a CTA take 16 keys each in turn with mma.sync m16n8k16, and everything a lane needs of a key it loads itself:
//   K: lane (g, t) = (lane / 4, lane % 4) holds key g's codes 64 i + 16 t .. + 15; the order of the products over hd is free as long as
//      q follows it, so four consecutive codes are the lane's B fragment of one k-step.
//   V: lane (g, t) holds codes 128 i + 16 g .. + 15 of keys 2t, 2t+1, 2t+8, 2t+9: as B fragments these are 16 output columns
//      (column g of tile b is hd index 128 i + 16 g + b), and the C fragments end up as 32 consecutive outputs a lane.
// So codes go from memory to fragments with 16-byte asynchronous copies into lane-private shared memory (a ring of stages a warp,
// no barriers, no bank conflicts) and a few integer instructions: code s eeee mmm becomes fp16 s 0eeee mmm 0000000, which is
// value * 2^-8, exactly, subnormals included; the 2^8 joins the scale of the scores and of the output.
// Keys are cut into chunks of kChunk over CTAs when a sequence is longer than that; partial results meet in the workspace and a
// second kernel joins them in chunk order, so that the result does not depend on timing.
#include "kv8.cuh"
#include "ptx.cuh"

namespace {

using namespace dc;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr uint32_t kTile = 16;       // keys a warp takes at a time; a page holds a whole number of tiles
constexpr uint32_t kMaxChunk = 32 * kWarps * kTile;   // a lane remembers the page of one of its warp's tiles: 32 tiles a warp
constexpr float kNone = -1e30f;      // running maximum of a row that has seen nothing
constexpr float kStep = 8.0f;        // the maximum follows only when it grows by more than 2^8
constexpr float kLog2e = 1.4426950408889634f;

template <int HD>
struct Shape {
    static constexpr int kStages = 3;
    static constexpr int kVec = 16 * HD / 16 / 32 * 2;              // 16-byte vectors a lane holds of a tile: K, then V
    static constexpr size_t kStage = static_cast<size_t>(kVec) * 512;   // bytes of a warp's stage
    static constexpr size_t kRing = kWarps * kStages * kStage;
    static constexpr size_t kQ = HD / 16 * 512;                     // q fragments: [k-step][lane] 16 bytes
    static constexpr size_t kBytes = kRing + kQ + 2 * 16 * 4;
    static_assert(kWarps * 16 * (HD + 2) * 4 <= kRing + kQ, "the warps' partial results reuse the ring");
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes in the high bytes of two halves -> two fp16 of value * 2^-8.
__device__ __forceinline__ uint32_t high_codes(uint32_t w) { return (w & 0x80008000u) | ((w >> 1) & 0x3f803f80u); }

// The rows of a tile: what the kernel and the join agree on.
struct Rows {
    uint32_t start, count, len;   // of the sequence: first packed row, rows, tokens
    bool ok;
};
__device__ __forceinline__ Rows rows_of(const dc_kv8_cache& c, const uint32_t* q_start, uint32_t j, uint32_t rows, uint32_t max_q) {
    Rows r;
    r.start = q_start[j];
    const uint32_t end = q_start[j + 1];
    r.len = c.lens[j];
    r.count = end - r.start;
    r.ok = end >= r.start && end <= rows && r.count <= max_q;
    return r;
}
// Tokens that row i of the sequence attends; *past is set where its position lies at or past the length.
__device__ __forceinline__ uint32_t visible(const Rows& r, const uint32_t* qpos, uint32_t i, bool* past) {
    if (!qpos) {
        const uint32_t behind = r.count - 1 - i;   // rows after this one
        if (behind >= r.len) {
            *past = r.len != 0u;
            return 0u;
        }
        return r.len - behind;
    }
    const uint32_t p = qpos[r.start + i];
    if (p == DC_KV8_NO_KEYS || r.len == 0u) return 0u;
    if (p >= r.len) *past = true;
    return min(p, r.len - 1) + 1;
}

struct Args {
    dc_kv8_cache c;   // k, v and the scales point at the layer
    const uint16_t* q;
    const float* gate;
    const uint32_t* q_start;
    const uint32_t* qpos;
    uint16_t* y;
    float* part;
    int* status;
    uint32_t rows, ldq, ldg, ldy, group, max_q, max_len, tiles, chunk, chunks;
    float scale;      // hd^-1/2 log2(e) 2^8
};

// o, normalised -> gate, 16 bits. 8 values of hd columns d .. d + 7.
template <typename Act>
__device__ __forceinline__ void store8(const Args& a, uint32_t row, uint32_t col, float (&o)[8]) {
    if (a.gate) {
        const float4 g0 = *reinterpret_cast<const float4*>(a.gate + static_cast<size_t>(row) * a.ldg + col);
        const float4 g1 = *reinterpret_cast<const float4*>(a.gate + static_cast<size_t>(row) * a.ldg + col + 4);
        const float g[8] = {g0.x, g0.y, g0.z, g0.w, g1.x, g1.y, g1.z, g1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] *= sigmoid_f(g[i]);
    }
    *reinterpret_cast<uint4*>(a.y + static_cast<size_t>(row) * a.ldy + col) =
        make_uint4(Act::pack(o[0], o[1]), Act::pack(o[2], o[3]), Act::pack(o[4], o[5]), Act::pack(o[6], o[7]));
}

// One CTA: 16 (row, head) pairs of a sequence's kv head over one chunk of its keys. FEW: at most 8 pairs, whose weights go in
// twice: rows 0..7 of the A operand hold them rounded to fp16 and rows 8..15 what the rounding left, so that the V product sees 22
// bits of each weight at no extra instruction of the tensor cores.
template <typename Act, int HD, bool FEW>
__global__ void __launch_bounds__(kThreads, HD == 128 ? 4 : 2) kv8_attn_kernel(const Args a) {
    using S = Shape<HD>;
    constexpr int kKVec = HD / 64;         // vectors of a key a lane holds
    constexpr int kVVec = HD / 128;
    extern __shared__ __align__(16) uint8_t smem[];
    uint8_t* ring = smem;
    uint4* qf = reinterpret_cast<uint4*>(smem + S::kRing);
    uint32_t* seen = reinterpret_cast<uint32_t*>(smem + S::kRing + S::kQ);   // [16] tokens that a pair attends
    float* rank = reinterpret_cast<float*>(seen + 16);                      // [16] power of two that a pair's q was divided by

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint32_t id = blockIdx.x;
    const uint32_t z = id % a.chunks;
    id /= a.chunks;
    const uint32_t tile_id = id;
    const uint32_t kvh = id % a.c.nkv;
    id /= a.c.nkv;
    const uint32_t mt = id % a.tiles, j = id / a.tiles;

    const Rows r = rows_of(a.c, a.q_start, j, a.rows, a.max_q);
    const bool reports = kvh == 0 && z == 0 && threadIdx.x == 0;
    if (!r.ok) {
        if (reports && mt == 0) kv8_flag(a.status, DC_STATUS_KV8_OFFSETS);
        return;
    }
    constexpr uint32_t kPairs = FEW ? 8 : 16;
    const uint32_t pair0 = mt * kPairs, pairs = r.count * a.group;
    if (pair0 >= pairs) return;
    if (r.len > a.max_len) {
        if (reports && mt == 0) kv8_flag(a.status, DC_STATUS_KV8_LENGTH);
        return;
    }
    if (warp == 0) {
        uint32_t n = 0;
        bool past = false;
        if (lane < static_cast<int>(kPairs) && pair0 + lane < pairs) n = visible(r, a.qpos, (pair0 + lane) / a.group, &past);
        if (lane < 16) seen[lane] = n;
        if (past && kvh == 0 && z == 0) kv8_flag(a.status, DC_STATUS_KV8_POSITION);
    }
    __syncthreads();
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < static_cast<int>(kPairs); ++i) most = max(most, seen[i]);
    const uint32_t key0 = z * a.chunk;
    if (z && key0 >= most) return;
    const uint32_t key1 = min(most, key0 + a.chunk);
    const uint32_t tiles = (key1 - key0 + kTile - 1) / kTile;                     // of the CTA
    const uint32_t mine = tiles > static_cast<uint32_t>(warp) ? (tiles - warp + kWarps - 1) / kWarps : 0u;   // of the warp: tile warp + kWarps i

    // lane i remembers page and scales of the warp's tile i
    uint64_t page_at = 0;
    float k_scale = 0.f, v_exp = 0.f;
    if (static_cast<uint32_t>(lane) < mine) {
        const uint32_t key = key0 + (warp + kWarps * lane) * kTile;
        uint32_t page = a.c.table[static_cast<size_t>(j) * a.c.max_pages + key / a.c.page_size];
        const bool inside = page < a.c.n_pages;
        if (!inside) {
            kv8_flag(a.status, DC_STATUS_KV8_PAGE);
            page = 0;
        }
        page_at = page * a.c.page_stride + kvh * a.c.head_stride + (key % a.c.page_size) * a.c.token_stride;
        k_scale = a.c.k_scale[static_cast<size_t>(page) * a.c.nkv + kvh];
        v_exp = kv8_log2i(a.c.v_scale[static_cast<size_t>(page) * a.c.nkv + kvh]);
        if (!inside) k_scale = __uint_as_float(0x7fffffffu);   // what attends it is NaN
    }

    const uint8_t* kc = static_cast<const uint8_t*>(a.c.k);
    const uint8_t* vc = static_cast<const uint8_t*>(a.c.v);
    const uint32_t my_ring = smem_u32(ring) + warp * (S::kStages * S::kStage) + lane * 16;
    auto fetch = [&](uint32_t i) {   // the warp's tile i; every lane runs this
        const uint64_t at = __shfl_sync(0xffffffffu, page_at, i & 31);
        uint32_t dst = my_ring + (i % S::kStages) * S::kStage;
        const uint8_t* ks = kc + at + 16 * t;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int v = 0; v < kKVec; ++v, dst += 512) cp16(dst, ks + (g + 8 * n) * a.c.token_stride + 64 * v);
        const uint8_t* vs = vc + at + 16 * g;
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
            for (int v = 0; v < kVVec; ++v, dst += 512) cp16(dst, vs + (2 * t + (p & 1) + 8 * (p >> 1)) * a.c.token_stride + 128 * v);
    };
#pragma unroll
    for (int i = 0; i + 1 < S::kStages; ++i) {
        if (static_cast<uint32_t>(i) < mine) fetch(i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // q as A fragments, in the order that the K codes lie in: k-step 4 v + w of lane (g, t) takes hd 64 v + 16 t + 4 w + {0, 2 | 1, 3}.
    // A bf16 row is first divided by a power of two that brings its largest magnitude to [2^14, 2^15): then its 8 bits fit fp16 but
    // for elements 2^-28 below it. fp16 rows go in as they are.
    for (uint32_t p = warp; p < 16; p += kWarps) {
        const bool on = p < kPairs && pair0 + p < pairs;
        const uint32_t row = r.start + (pair0 + p) / a.group, h = kvh * a.group + (pair0 + p) % a.group;
        const uint16_t* src = a.q + static_cast<size_t>(row) * a.ldq + static_cast<size_t>(h) * HD;
        constexpr int kWords = HD / 128;   // 8-byte pieces a lane holds: piece lane + 32 i is hd 4 (lane + 32 i) ..
        uint2 x[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) x[i] = on ? *reinterpret_cast<const uint2*>(src + 4 * (lane + 32 * i)) : make_uint2(0, 0);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < kWords; ++i) top = __vmaxu2(top, __vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu));
        top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
        float up = 1.f;
        if (Act::kUmmaFormat == 1) {
            const uint32_t e = top >> 7;   // exponent field of the largest
            // 2^(e - 127) -> 2^14; fields beyond 1 .. 254 (zeros, subnormals, infinities) take the nearest
            const int shift = min(max(static_cast<int>(e), 1), 254) - 127 - 14;
            const int half = shift / 2;   // two factors: 2^-shift alone may pass fp32's exponents
            const float down = kv8_exp2i(-half), rest_down = kv8_exp2i(-(shift - half));
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                x[i].x = ActF16::pack(Act::lo(x[i].x) * down * rest_down, Act::hi(x[i].x) * down * rest_down);
                x[i].y = ActF16::pack(Act::lo(x[i].y) * down * rest_down, Act::hi(x[i].y) * down * rest_down);
            }
            up = kv8_exp2i(half) * kv8_exp2i(shift - half);
        }
        if (!(Act::one(static_cast<uint16_t>(top)) <= 3.4028235e38f)) up = __uint_as_float(0x7fffffffu);   // a row that is not finite: NaN
        if (lane == 0) rank[p] = up;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const uint32_t hd = 4 * (lane + 32 * i), step = hd / 64 * 4 + hd % 16 / 4, to = hd % 64 / 16;   // to: t of the lane it belongs to
            uint32_t* f = reinterpret_cast<uint32_t*>(qf + step * 32 + (p & 7) * 4 + to);
            f[p >> 3] = (x[i].x & 0xffffu) | (x[i].y << 16);                 // hd + 0, hd + 2: k = 2t, 2t + 1
            f[2 + (p >> 3)] = (x[i].x >> 16) | (x[i].y & 0xffff0000u);       // hd + 1, hd + 3: k = 2t + 8, 2t + 9
        }
    }
    __syncthreads();

    const uint32_t see0 = seen[g], see1 = seen[FEW ? g : g + 8];
    const float mul0 = a.scale * rank[g], mul1 = FEW ? 0.f : a.scale * rank[g + 8];
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m0 = kNone, m1 = kNone, l0 = 0.f, l1 = 0.f;

    for (uint32_t i = 0; i < mine; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
        const uint8_t* at = ring + warp * (S::kStages * S::kStage) + (i % S::kStages) * S::kStage + lane * 16;
        float s[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
            for (int v = 0; v < kKVec; ++v) {
                const uint4 x = *reinterpret_cast<const uint4*>(at + (n * kKVec + v) * 512);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint4 f = qf[(4 * v + e) * 32 + lane];
                    mma_f16(s[n], f.x, f.y, f.z, f.w, high_codes(w[e] << 8), high_codes(w[e]));
                }
            }
        }
        const float ks = __shfl_sync(0xffffffffu, k_scale, i & 31);
        float ve = __shfl_sync(0xffffffffu, v_exp, i & 31);
        const float back = isnan(ve) ? 1.f : kv8_exp2i(max(-126, min(127, -static_cast<int>(ve))));   // 2^-e_v; a NaN reaches the sum through the weights
        const uint32_t key = key0 + (warp + kWarps * i) * kTile + 2 * t;
        const float c0 = mul0 * ks, c1 = mul1 * ks;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[n][e] = key + 8 * n + e < see0 ? fmaf(s[n][e], c0, ve) : -INFINITY;
                if (!FEW) s[n][2 + e] = key + 8 * n + e < see1 ? fmaf(s[n][2 + e], c1, ve) : -INFINITY;
            }
        const float top0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        const float top1 = FEW ? -INFINITY : fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
        if (__any_sync(0xffffffffu, top0 > m0 + kStep || (!FEW && top1 > m1 + kStep))) {
            // the four lanes of a row agree on the new maximum; rows whose maximum stays put scale by 1
            float n0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 1));
            n0 = fmaxf(m0, fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, 2)));
            const float by0 = ex2(m0 - n0);
            m0 = n0;
            l0 *= by0;
            float by1 = by0;
            if (!FEW) {
                float n1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 1));
                n1 = fmaxf(m1, fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, 2)));
                by1 = ex2(m1 - n1);
                m1 = n1;
                l1 *= by1;
            }
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) {
                o[d][0] *= by0;
                o[d][1] *= by0;
                o[d][2] *= by1;
                o[d][3] *= by1;
            }
        }
        float p[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                p[n][e] = ex2(s[n][e] - m0);
                l0 = fmaf(p[n][e], back, l0);
                if (!FEW) {
                    p[n][2 + e] = ex2(s[n][2 + e] - m1);
                    l1 = fmaf(p[n][2 + e], back, l1);
                }
            }
        const uint32_t a0 = ActF16::pack(p[0][0], p[0][1]), a2 = ActF16::pack(p[1][0], p[1][1]);
        uint32_t a1, a3;
        if (FEW) {
            a1 = ActF16::pack(p[0][0] - ActF16::lo(a0), p[0][1] - ActF16::hi(a0));
            a3 = ActF16::pack(p[1][0] - ActF16::lo(a2), p[1][1] - ActF16::hi(a2));
        } else {
            a1 = ActF16::pack(p[0][2], p[0][3]);
            a3 = ActF16::pack(p[1][2], p[1][3]);
        }
#pragma unroll
        for (int v = 0; v < kVVec; ++v) {
            uint32_t x[4][4];
#pragma unroll
            for (int p4 = 0; p4 < 4; ++p4) {
                const uint4 u = *reinterpret_cast<const uint4*>(at + (2 * kKVec + p4 * kVVec + v) * 512);
                x[p4][0] = u.x, x[p4][1] = u.y, x[p4][2] = u.z, x[p4][3] = u.w;
            }
#pragma unroll
            for (int b = 0; b < 16; ++b) {
                // byte b % 4 of two keys' words into the high bytes of two halves
                const uint32_t pick = ((b & 3) << 4) | ((4 + (b & 3)) << 12);
                mma_f16(o[16 * v + b], a0, a1, a2, a3, high_codes(__byte_perm(x[0][b >> 2], x[1][b >> 2], pick)),
                        high_codes(__byte_perm(x[2][b >> 2], x[3][b >> 2], pick)));
            }
        }
        if (i + S::kStages - 1 < mine) fetch(i + S::kStages - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

    // the four lanes of a row add their sums; the warps' partial results meet in shared memory
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    __syncthreads();   // the ring and the q fragments are free
    constexpr int kLd = HD + 2;
    float* mine_at = reinterpret_cast<float*>(smem) + warp * (kPairs * kLd);
    if (t == 0) {
        mine_at[g * kLd + HD] = m0;
        mine_at[g * kLd + HD + 1] = l0;
        if (!FEW) {
            mine_at[(g + 8) * kLd + HD] = m1;
            mine_at[(g + 8) * kLd + HD + 1] = l1;
        }
    }
#pragma unroll
    for (int v = 0; v < kVVec; ++v)
#pragma unroll
        for (int b = 0; b < 16; ++b) {
            const int d = 128 * v + 32 * t + b;
            const float (&x)[4] = o[16 * v + b];
            mine_at[g * kLd + d] = FEW ? x[0] + x[2] : x[0];
            mine_at[g * kLd + d + 16] = FEW ? x[1] + x[3] : x[1];
            if (!FEW) {
                mine_at[(g + 8) * kLd + d] = x[2];
                mine_at[(g + 8) * kLd + d + 16] = x[3];
            }
        }
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(smem);
    const bool whole = most <= a.chunk;   // this CTA has seen every key
    for (uint32_t e = threadIdx.x; e < kPairs * (HD / 8); e += kThreads) {
        const uint32_t p = e / (HD / 8), d = e % (HD / 8) * 8;
        if (pair0 + p >= pairs) continue;
        float m = kNone, l = 0.f, x[8] = {};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) m = fmaxf(m, all[(w * kPairs + p) * kLd + HD]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float* from = all + (w * kPairs + p) * kLd;
            const float by = ex2(from[HD] - m);
            l = fmaf(from[HD + 1], by, l);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(from[d + i], by, x[i]);
        }
        if (whole) {
            const float by = l == 0.f ? 0.f : 256.f / l;   // a row that attends nothing
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= by;
            store8<Act>(a, r.start + (pair0 + p) / a.group, (kvh * a.group + (pair0 + p) % a.group) * HD + d, x);
        } else {
            float* to = a.part + ((static_cast<size_t>(tile_id) * a.chunks + z) * kPairs + p) * (HD + 4);
            *reinterpret_cast<float4*>(to + d) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(to + d + 4) = make_float4(x[4], x[5], x[6], x[7]);
            if (d == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(m, l);
        }
    }
}

// Joins the chunks of a tile's pairs, in chunk order. One CTA a tile; tiles that one chunk held have written their rows already.
template <typename Act, int HD>
__global__ void __launch_bounds__(256) kv8_join_kernel(const Args a, uint32_t per_tile) {
    uint32_t id = blockIdx.x;
    const uint32_t tile_id = id, kvh = id % a.c.nkv;
    id /= a.c.nkv;
    const uint32_t mt = id % a.tiles, j = id / a.tiles;
    const Rows r = rows_of(a.c, a.q_start, j, a.rows, a.max_q);
    if (!r.ok || r.len > a.max_len) return;
    const uint32_t pair0 = mt * per_tile, pairs = r.count * a.group;
    if (pair0 >= pairs) return;
    uint32_t most = 0;
    bool past = false;
    if ((threadIdx.x & 31) < per_tile && pair0 + (threadIdx.x & 31) < pairs) most = visible(r, a.qpos, (pair0 + (threadIdx.x & 31)) / a.group, &past);
    most = __reduce_max_sync(0xffffffffu, most);
    if (most <= a.chunk) return;
    const uint32_t chunks = (most + a.chunk - 1) / a.chunk;
    const size_t step = static_cast<size_t>(per_tile) * (HD + 4);
    for (uint32_t e = threadIdx.x; e < per_tile * (HD / 8); e += 256) {
        const uint32_t p = e / (HD / 8), d = e % (HD / 8) * 8;
        if (pair0 + p >= pairs) continue;
        const float* from = a.part + (static_cast<size_t>(tile_id) * a.chunks * per_tile + p) * (HD + 4);
        float m = kNone, l = 0.f, x[8] = {};
        for (uint32_t z = 0; z < chunks; ++z) m = fmaxf(m, from[z * step + HD]);
        for (uint32_t z = 0; z < chunks; ++z) {
            const float2 ml = *reinterpret_cast<const float2*>(from + z * step + HD);
            const float4 u = *reinterpret_cast<const float4*>(from + z * step + d), w = *reinterpret_cast<const float4*>(from + z * step + d + 4);
            const float by = ex2(ml.x - m), v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
            l = fmaf(ml.y, by, l);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(v[i], by, x[i]);
        }
        const float by = l == 0.f ? 0.f : 256.f / l;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= by;
        store8<Act>(a, r.start + (pair0 + p) / a.group, (kvh * a.group + (pair0 + p) % a.group) * HD + d, x);
    }
}

// How a call is cut: tiles of `pairs` (row, head) pairs, chunks of `chunk` keys.
struct Cut {
    uint32_t pairs, tiles, max_len, chunk, chunks;
    uint64_t ctas;
};
Cut cut_of(const dc_ctx* ctx, const dc_kv8_cache* c, uint32_t nq, uint32_t max_q, uint32_t max_len) {
    Cut t;
    const uint32_t group = nq / c->nkv;
    const uint64_t pairs = static_cast<uint64_t>(max_q) * group;
    t.pairs = pairs <= 8 ? 8 : 16;
    t.tiles = static_cast<uint32_t>((pairs + t.pairs - 1) / t.pairs);
    const uint32_t cap = c->max_pages * c->page_size;
    const uint32_t len = max_len == 0 || max_len > cap ? cap : max_len;
    const uint64_t whole = static_cast<uint64_t>(c->n_seqs) * c->nkv * t.tiles;
    // Chunks as long as they can be while there are about six CTAs an SM to balance the load with, from 256 to kMaxChunk keys.
    const uint64_t want = (static_cast<uint64_t>(ctx->sm_count) * 6 + whole - 1) / whole;
    uint64_t chunk = (len + want - 1) / want;
    chunk = (chunk + 127) / 128 * 128;
    t.chunk = static_cast<uint32_t>(chunk < 256 ? 256 : chunk > kMaxChunk ? kMaxChunk : chunk);
    t.max_len = len;
    t.chunks = (len + t.chunk - 1) / t.chunk;
    t.ctas = whole * t.chunks;
    return t;
}
size_t part_bytes(const dc_kv8_cache* c, const Cut& t) {
    if (t.chunks <= 1) return 0;
    return static_cast<size_t>(t.ctas) * t.pairs * (c->hd + 4) * sizeof(float);
}

typedef void (*attn_fn)(const Args);
template <typename Act>
attn_fn pick(uint32_t hd, bool few) {
    if (hd == 128) return few ? kv8_attn_kernel<Act, 128, true> : kv8_attn_kernel<Act, 128, false>;
    return few ? kv8_attn_kernel<Act, 256, true> : kv8_attn_kernel<Act, 256, false>;
}

}  // namespace

int dc_kv8_attention_warm(dc_ctx* ctx) {
    static bool set[16] = {};
    if (set[ctx->device & 15]) return DC_OK;
    for (int i = 0; i < 8; ++i) {
        const uint32_t hd = i & 1 ? 256 : 128;
        const attn_fn f = i & 4 ? pick<dc::ActF16>(hd, i & 2) : pick<dc::ActBF16>(hd, i & 2);
        const int bytes = static_cast<int>(hd == 128 ? Shape<128>::kBytes : Shape<256>::kBytes);
        const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return dc_fail(ctx, DC_CUDA_ERROR, "kv8_attention: cannot opt in to %d bytes of shared memory: %s", bytes, cudaGetErrorString(e));
    }
    set[ctx->device & 15] = true;
    return DC_OK;
}

extern "C" size_t dc_kv8_attention_scratch_bytes(dc_ctx* ctx, const dc_kv8_cache* cache, uint32_t nq, uint32_t max_q, uint32_t max_len) {
    if (!ctx || dc_kv8_check(cache, nullptr, 0) != DC_OK || nq == 0 || nq % cache->nkv || max_q == 0) return 0;
    return part_bytes(cache, cut_of(ctx, cache, nq, max_q, max_len));
}

extern "C" int dc_kv8_attention(dc_ctx* ctx, void* stream, const dc_kv8_cache* cache, uint32_t layer, const void* q, const float* gate,
                                const uint32_t* q_start, const uint32_t* qpos, void* y, uint32_t rows, uint32_t ldq, uint32_t ldg, uint32_t ldy,
                                uint32_t nq, uint32_t max_q, uint32_t max_len) {
    if (!ctx) return DC_INVALID_ARG;
    int rc = dc_kv8_require(ctx, "kv8_attention", cache);
    if (rc != DC_OK) return rc;
    DC_REQUIRE(ctx, q && q_start && y, "kv8_attention: null operand");
    DC_REQUIRE(ctx, layer < cache->layers, "kv8_attention: layer %u of %u", layer, cache->layers);
    DC_REQUIRE(ctx, nq >= 1 && nq % cache->nkv == 0, "kv8_attention: %u query heads over %u kv heads", nq, cache->nkv);
    if (nq / cache->nkv > 16) return dc_fail(ctx, DC_UNSUPPORTED, "kv8_attention: %u query heads per kv head (at most 16)", nq / cache->nkv);
    const uint64_t width = static_cast<uint64_t>(nq) * cache->hd;
    DC_REQUIRE(ctx, ldq >= width && ldq % 8 == 0 && ldy >= width && ldy % 8 == 0, "kv8_attention: ldq = %u, ldy = %u must cover nq * hd = %llu and be multiples of 8",
               ldq, ldy, static_cast<unsigned long long>(width));
    DC_REQUIRE(ctx, !gate || (ldg >= width && ldg % 4 == 0 && reinterpret_cast<uintptr_t>(gate) % 16 == 0),
               "kv8_attention: ldg = %u must cover the gate columns and be a multiple of 4, gate 16-byte aligned", ldg);
    DC_REQUIRE(ctx, reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(y) % 16 == 0, "kv8_attention: q and y must be 16-byte aligned");
    if (rows == 0 || max_q == 0) return DC_OK;   // no rows: nothing to write
    const uint32_t most = max_q < rows ? max_q : rows;
    const dc_device_scope scope(ctx);
    const Cut t = cut_of(ctx, cache, nq, most, max_len);
    DC_REQUIRE(ctx, t.ctas < 0x7fffffffull, "kv8_attention: %llu CTAs: fewer rows or sequences a call", static_cast<unsigned long long>(t.ctas));
    Args a;
    a.c = *cache;
    a.c.k = static_cast<uint8_t*>(cache->k) + layer * cache->layer_stride;
    a.c.v = static_cast<uint8_t*>(cache->v) + layer * cache->layer_stride;
    a.c.k_scale = cache->k_scale + static_cast<size_t>(layer) * cache->n_pages * cache->nkv;
    a.c.v_scale = cache->v_scale + static_cast<size_t>(layer) * cache->n_pages * cache->nkv;
    a.part = nullptr;
    if (t.chunks > 1) {
        void* ws = nullptr;
        if ((rc = dc_get_workspace(ctx, part_bytes(cache, t), "kv8_attention", &ws)) != DC_OK) return rc;
        a.part = static_cast<float*>(ws);
    }
    if ((rc = dc_kv8_attention_warm(ctx)) != DC_OK) return rc;
    a.q = static_cast<const uint16_t*>(q);
    a.gate = gate;
    a.q_start = q_start;
    a.qpos = qpos;
    a.y = static_cast<uint16_t*>(y);
    a.status = ctx->status_dev;
    a.rows = rows, a.ldq = ldq, a.ldg = ldg, a.ldy = ldy, a.group = nq / cache->nkv, a.max_q = most, a.max_len = t.max_len;
    a.tiles = t.tiles, a.chunk = t.chunk, a.chunks = t.chunks;
    a.scale = 256.f * kLog2e / sqrtf(static_cast<float>(cache->hd));
    const bool f16 = ctx->act_dtype == DC_ACT_F16;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const attn_fn f = f16 ? pick<dc::ActF16>(cache->hd, t.pairs == 8) : pick<dc::ActBF16>(cache->hd, t.pairs == 8);
    f<<<static_cast<uint32_t>(t.ctas), kThreads, cache->hd == 128 ? Shape<128>::kBytes : Shape<256>::kBytes, s>>>(a);
    if ((rc = dc_check_launch(ctx, "kv8_attention")) != DC_OK || t.chunks == 1) return rc;
    auto join = cache->hd == 128 ? (f16 ? kv8_join_kernel<dc::ActF16, 128> : kv8_join_kernel<dc::ActBF16, 128>)
                                 : (f16 ? kv8_join_kernel<dc::ActF16, 256> : kv8_join_kernel<dc::ActBF16, 256>);
    join<<<static_cast<uint32_t>(t.ctas / t.chunks), 256, 0, s>>>(a, t.pairs);
    return dc_check_launch(ctx, "kv8_attention (join)");
}
