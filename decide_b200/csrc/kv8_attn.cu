// dc_kv8_attention: causal GQA attention over one layer of the paged 8-bit K/V cache.
//
// The mathematics. With codes k', v' and page scales a = 2^e_k, b = 2^e_v (per page and kv head), row r of head h has scores
// s_j = a_j (q . k'_j) hd^-1/2 and o = sum_j softmax(s)_j b_j v'_j. Taking the V scale into the exponent, with t_j = s_j log2(e) + e_v(j):
//     o = sum_j 2^(t_j - m) v'_j / sum_j 2^(t_j - m) 2^-e_v(j),    m the largest t_j up to a factor,
// so that one running maximum serves both sums, the weights of the V product are relative to the row's largest TERM, and no code is
// ever scaled: codes go into the tensor cores as fp16, exactly. The V product takes the weights in fp16, whose range below the largest
// term is what kKv8Below is about: a term under 2^-32 of it drops out of the product. The total is fp32.
//
// K/V bytes bound it when there are few rows. A CTA takes up to 8 NT (query row, head of the group) pairs that share a kv head's codes; its
// warps take 16 keys each in turn with mma.sync m16n8k16, codes as the A operand (so that 16 keys, or 16 columns of V, fill it, and
// a tile of 8 pairs costs HD / 8 MMAs), and everything a lane needs of a key it loads itself:
//   S^T = K Q^T: lane (g, t) = (lane / 4, lane % 4) holds codes 64 i + 16 t .. + 15 of keys g and g + 8; the order of the products over hd
//      is free as long as q follows it, so four consecutive codes are the lane's share of one k-step.
//   O^T = V^T P^T: lane (g, t) holds codes 128 i + 16 g .. + 15 of keys 2t, 2t+1, 2t+8, 2t+9: as A fragments these are 16 columns,
//      two to a tile, and the C fragments end up as 16 consecutive outputs of a pair. P^T comes from the C fragments of S^T by
//      movmatrix.
// Codes go from memory to fragments with 16-byte asynchronous copies of whole rows into a ring of stages that belongs to the warp (no CTA
// barriers), 16-byte reads, a byte permutation for V and one conversion for two codes. A stage holds 16 rows of K, then of V; the
// 16-byte pieces of each 128 bytes of a row lie at piece ^ 4 (row & 1) for K and piece ^ (row & 6) for V: a row is written in
// one pass over the banks, and the eight lanes of a read's phase, two keys by four pieces of K or four keys by two of V, meet all 32
// banks. (Pieces lying where their lanes read them were written four passes a row: 201 instead of 68 a tile, which bound the kernel.)
// Codes that append has written are finite; what lies behind a sequence's last token, or has not been written since the sequence
// grew, may be the code for NaN, and a weight of zero would not hide it: V codes that no row of the tile attends are replaced by zeros.
// Keys are cut into chunks over CTAs; partial results meet in the workspace, and the CTA of a tile that finishes last (a counter tells)
// joins them in chunk order, so that the result does not depend on timing.
// Measured on the device, 8 kv heads of 128, 4 queries each: one token over 131,071 keys 51 us (268 MB, 5.3 TB/s); a token for each of 64
// sequences of 576 to 2,307 42.6 us (186 MB, 4.4 TB/s; in the loop 5.6); one over 603 keys 6.8 us. A tile of 16 keys costs a warp 275
// instructions (466 with the keys as the B operand, half of whose 16 rows of pairs were empty, and codes turned by integer steps).
#include <cmath>
#include "kv8_attn.cuh"
#include "ptx.cuh"

namespace {

using namespace dc;

constexpr uint32_t kTile = 16;       // keys a warp takes at a time; a page holds a whole number of tiles

template <int HD, int NT>
struct Shape {
    static constexpr int kWarps = HD * NT <= 256 && HD == 128 ? 8 : 4;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kStages = 3;
    static constexpr int kPairs = 8 * NT;
    static constexpr int kVec = HD / 16;                            // 16-byte vectors a lane holds of a tile: half K, half V
    static constexpr size_t kStage = static_cast<size_t>(kVec) * 512;   // bytes of a warp's stage
    static constexpr size_t kRing = kWarps * kStages * kStage;
    static constexpr int kLd = HD + 4;                              // floats of a pair's partial result: sums, maximum, total
    static constexpr size_t kParts = static_cast<size_t>(kWarps) * kPairs * kLd * 4;   // the warps' results reuse the ring
    static constexpr size_t kQ = kRing > kParts ? kRing : kParts;   // offset of the q fragments: [k-step][8 pairs][lane] 8 bytes
    static constexpr size_t kSeen = kQ + static_cast<size_t>(HD / 16) * NT * 256;
    static constexpr size_t kBytes = kSeen + 2 * kPairs * 4 + 16;
    static constexpr int kBlocks = (HD * NT <= 256 ? 16 : HD * NT <= 384 ? 12 : 8) / kWarps;   // CTAs an SM that registers and shared memory leave room for
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit elements held as C fragments (lane (g, t): row g, columns 2t, 2t + 1).
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// A weight as the total counts it: rounded, as the V product takes it, so that what rounding does to a row that one key dominates cancels;
// but exact where fp16 runs out of bits (below 2^-14), since a key whose page has a small V scale may weigh much in the total and
// little in the product.
__device__ __forceinline__ float kv8_total(float exact, float rounded) { return exact >= 6.103515625e-05f ? rounded : exact; }

// One CTA: 8 NT (row, head) pairs of a sequence's kv head over one chunk of its keys.
template <typename Act, int HD, int NT>
__global__ void __launch_bounds__(Shape<HD, NT>::kThreads, Shape<HD, NT>::kBlocks) kv8_attn_kernel(const Kv8Args a) {
    using S = Shape<HD, NT>;
    constexpr int kWarps = S::kWarps, kThreads = S::kThreads;
    constexpr int kKVec = HD / 64;         // vectors of a key a lane holds
    constexpr int kVVec = HD / 128;
    constexpr uint32_t kPairs = S::kPairs;
    extern __shared__ __align__(1024) uint8_t smem[];
    uint2* qf = reinterpret_cast<uint2*>(smem + S::kQ);
    uint32_t* seen = reinterpret_cast<uint32_t*>(smem + S::kSeen);   // tokens that a pair attends
    float* rank = reinterpret_cast<float*>(seen + kPairs);           // power of two that a pair's q was divided by

    kv8_begin();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint32_t id = blockIdx.x;
    const uint32_t z = id % a.chunks;
    id /= a.chunks;
    const uint32_t tile_id = id;
    const uint32_t kvh = id % a.c.nkv;
    id /= a.c.nkv;
    const uint32_t mt = id % a.tiles, j = id / a.tiles;

    // The pages of the warp's tiles warp + kWarps i: lane i remembers that of tile i, 32 tiles at a time, and its scales. Where the last key
    // is not known yet, the table is read ahead of it (never past its row).
    const uint32_t key0 = z * a.chunk;
    const uint32_t* table = a.c.table + static_cast<size_t>(j) * a.c.max_pages;
    auto column = [&](uint32_t i) { return (key0 + (warp + kWarps * i) * kTile) >> a.page_shift; };
    uint32_t page_ahead = column(lane) < a.c.max_pages ? table[column(lane)] : 0u;
    const Kv8Rows r = kv8_rows(a.c, a.q_start, j, a.rows, a.max_q);
    const bool reports = kvh == 0 && z == 0 && threadIdx.x == 0;
    if (!r.ok) {
        if (reports && mt == 0) kv8_flag(a.status, DC_STATUS_KV8_OFFSETS);
        return;
    }
    const uint32_t pair0 = mt * kPairs, pairs = r.count * a.group;
    if (pair0 >= pairs) return;
    if (r.len > a.max_len) {
        if (reports && mt == 0) kv8_flag(a.status, DC_STATUS_KV8_LENGTH);
        return;
    }
    uint32_t n = 0;   // every warp: lane p looks at pair p
    const bool on = lane < static_cast<int>(kPairs) && pair0 + lane < pairs;
    {
        bool past = false;
        if (on) n = kv8_visible(r, a.qpos, kv8_row_of(a, pair0 + lane), &past);
        if (past && kvh == 0 && z == 0 && warp == 0) kv8_flag(a.status, DC_STATUS_KV8_POSITION);
    }
    const uint32_t most = __reduce_max_sync(0xffffffffu, n), least = __reduce_min_sync(0xffffffffu, on ? n : 0xffffffffu);
    if (z && key0 >= most) return;
    if (warp == 0 && lane < static_cast<int>(kPairs)) seen[lane] = n;
    const uint32_t key1 = min(most, key0 + a.chunk);
    const uint32_t tiles = (key1 - key0 + kTile - 1) / kTile;                     // of the CTA
    const uint32_t mine = tiles > static_cast<uint32_t>(warp) ? (tiles - warp + kWarps - 1) / kWarps : 0u;   // of the warp: tile warp + kWarps i

    uint64_t page_at = 0;                   // of the 32 tiles being fetched
    float next_k = 0.f, next_v = 0.f;       // their scales
    auto turn = [&](uint32_t i) {           // to tiles i .. i + 31
        const uint32_t mine_i = i + lane, key = key0 + (warp + kWarps * mine_i) * kTile;
        if (mine_i < mine) {
            uint32_t page = i ? table[column(mine_i)] : page_ahead;
            const bool inside = page < a.c.n_pages;
            if (!inside) {
                kv8_flag(a.status, DC_STATUS_KV8_PAGE);
                page = 0;
            }
            page_at = page * a.c.page_stride + kvh * a.c.head_stride + (key & (a.c.page_size - 1)) * a.c.token_stride;
            next_k = a.c.k_scale[static_cast<size_t>(page) * a.c.nkv + kvh];
            next_v = a.c.v_scale[static_cast<size_t>(page) * a.c.nkv + kvh];
            if (!inside) next_k = __uint_as_float(0x7fffffffu);   // what attends it is NaN (and page 0's V codes are not used)
        }
    };

    // A warp copies kRows rows of HD codes an instruction.
    constexpr int kRows = 512 / HD, kPieces = HD / 16;
    const uint32_t token = static_cast<uint32_t>(a.c.token_stride);
    const uint32_t fill_row = lane / kPieces, piece = lane % kPieces;
    const uint8_t* kc = static_cast<const uint8_t*>(a.c.k) + fill_row * token + 16 * piece;
    const uint8_t* vc = static_cast<const uint8_t*>(a.c.v) + fill_row * token + 16 * piece;
    const uint8_t* ring = smem + warp * (S::kStages * S::kStage);
    const uint32_t fill_k = smem_u32(ring) + fill_row * HD + 16 * (piece ^ (4 * (fill_row & 1))), fill_v = smem_u32(ring) + 16 * HD + fill_row * HD + 16 * (piece ^ (fill_row & 6));
    auto fetch = [&](uint32_t i, uint32_t stage) {   // the warp's tile i; every lane runs this
        if (i % 32 == 0) turn(i);
        const uint64_t at = __shfl_sync(0xffffffffu, page_at, i % 32);
        const uint32_t to = stage * static_cast<uint32_t>(S::kStage);
        const uint8_t *ks = kc + at, *vs = vc + at;
#pragma unroll
        for (int n = 0; n < 16 / kRows; ++n, ks += kRows * token, vs += kRows * token) {
            cp16(fill_k + to + n * 512, ks);
            cp16((fill_v ^ (16 * (n * kRows & 6))) + to + n * 512, vs);
        }
    };
#pragma unroll
    for (int i = 0; i + 1 < S::kStages; ++i) {
        if (static_cast<uint32_t>(i) < mine) fetch(i, i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // q as B fragments, in the order that the K codes lie in: k-step 4 v + w of lane (g, t) takes hd 64 v + 16 t + 4 w + {0, 1 | 2, 3}, 8 bytes
    // of q as they are.
    for (uint32_t p = warp; p < kPairs; p += kWarps) {
        const bool there = pair0 + p < pairs;
        const uint32_t of = kv8_row_of(a, pair0 + p), row = r.start + of, h = kvh * a.group + pair0 + p - of * a.group;
        const uint16_t* src = a.q + static_cast<size_t>(row) * a.ldq + static_cast<size_t>(h) * HD;
        constexpr int kWords = HD / 128;   // 8-byte pieces a lane holds: piece lane + 32 i is hd 4 (lane + 32 i) ..
        uint2 x[kWords];
#pragma unroll
        for (int i = 0; i < kWords; ++i) x[i] = there ? *reinterpret_cast<const uint2*>(src + 4 * (lane + 32 * i)) : make_uint2(0, 0);
        const float up = kv8_query_row<Act, kWords>(x, kv8_query_top<kWords>(x));
        if (lane == 0) rank[p] = up;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const uint32_t hd = 4 * (lane + 32 * i), step = hd / 64 * 4 + hd % 16 / 4, to = hd % 64 / 16;   // to: t of the lane it belongs to
            qf[(step * NT + (p >> 3)) * 32 + (p & 7) * 4 + to] = x[i];
        }
    }
    __syncthreads();

    // pairs 8 n + 2 t and + 1 of each tile of pairs: the columns of this lane's C fragments
    float mul[NT][2], m[NT][2], l[NT][2];
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            mul[b][e] = rank[8 * b + 2 * t + e];
            m[b][e] = kKv8None;
            l[b][e] = 0.f;
        }
    constexpr bool kKeepQ = NT * HD <= 128;   // q fragments in registers where there is room
    uint2 q_kept[kKeepQ ? HD / 16 : 1];
    if (kKeepQ) {
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) q_kept[kKeepQ ? i : 0] = qf[i * 32 + lane];
    }
    float o[NT][HD / 16][4];
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int d = 0; d < HD / 16; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[b][d][e] = 0.f;

    const uint32_t read_k0 = g * HD + 16 * (t + 4 * (g & 1)), read_k1 = read_k0 ^ 64, read_v = 16 * HD + 2 * t * HD + 16 * (g ^ (2 * t));
    uint32_t stage = 0;
    float k_scale = 0.f, v_scale = 0.f;   // of the 32 tiles being worked on
    for (uint32_t i = 0; i < mine; ++i) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 2) : "memory");
        __syncwarp();   // all lanes' copies of this stage have landed, and all have read the stage that is filled next
        if (i % 32 == 0) k_scale = next_k, v_scale = next_v;
        const uint8_t* at = ring + stage * S::kStage;
        const uint32_t key = key0 + (warp + kWarps * i) * kTile;
        float s[NT][4];
#pragma unroll
        for (int b = 0; b < NT; ++b) s[b][0] = s[b][1] = s[b][2] = s[b][3] = 0.f;
#pragma unroll
        for (int v = 0; v < kKVec; ++v) {
            const uint8_t* from = at + (v & 1 ? read_k1 : read_k0) + 128 * (v >> 1);
            const uint4 x = *reinterpret_cast<const uint4*>(from), y = *reinterpret_cast<const uint4*>(from + 8 * HD);
            const uint32_t w0[4] = {x.x, x.y, x.z, x.w}, w1[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t a0 = low_codes(w0[e]), a1 = low_codes(w1[e]), a2 = high_codes(w0[e]), a3 = high_codes(w1[e]);
#pragma unroll
                for (int b = 0; b < NT; ++b) {
                    const uint2 f = kKeepQ ? q_kept[kKeepQ ? 4 * v + e : 0] : qf[((4 * v + e) * NT + b) * 32 + lane];
                    mma_f16(s[b], a0, a1, a2, a3, f.x, f.y);
                }
            }
        }
        // (hd^-1/2 goes with the K scale: with q's power of two, 2^-140 for the smallest of bf16, it would leave fp32's normal numbers)
        const float ks = a.scale * __shfl_sync(0xffffffffu, k_scale, i % 32), ve = kv8_log2i(__shfl_sync(0xffffffffu, v_scale, i % 32));
        const float back = isnan(ve) ? 1.f : kv8_exp2i(max(-126, min(127, -static_cast<int>(ve))));   // 2^-e_v; a NaN reaches the sum through the weights
        bool grow = false;
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float by = mul[b][e] * ks;
                s[b][e] = fmaf(s[b][e], by, ve);
                s[b][2 + e] = fmaf(s[b][2 + e], by, ve);
            }
        if (key + kTile > least) {   // some pair does not see all of the tile
#pragma unroll
            for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t see = seen[8 * b + 2 * t + e];
                    if (key + g >= see) s[b][e] = -INFINITY;
                    if (key + g + 8 >= see) s[b][2 + e] = -INFINITY;
                }
        }
#pragma unroll
        for (int b = 0; b < NT; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) grow |= fmaxf(s[b][e], s[b][2 + e]) > m[b][e] + kKv8Step;
        if (__any_sync(0xffffffffu, grow)) {
            // the eight lanes of a pair agree on the new maximum; pairs whose maximum stays put scale by 1
#pragma unroll
            for (int b = 0; b < NT; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(s[b][e], s[b][2 + e]);
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                    top = fmaxf(m[b][e], fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)) - kKv8Below);
                    const float by = ex2(m[b][e] - top);
                    m[b][e] = top;
                    l[b][e] *= by;
#pragma unroll
                    for (int d = 0; d < HD / 16; ++d) {
                        o[b][d][e] *= by;
                        o[b][d][2 + e] *= by;
                    }
                }
        }
        // The weights as B fragments. One set of eight pairs goes in twice, rounded to fp16 and what that left (22 bits down to 2^-10 of the row's
        // largest term, one less for each 2^-1 below, for eight more MMAs that memory hides); two sets go in once, and the total adds them as they go in (kv8_total).
        constexpr bool kTwice = NT == 1;
        uint32_t p0[NT], p1[NT], q0 = 0, q1 = 0;
#pragma unroll
        for (int b = 0; b < NT; ++b) {
            const float w00 = ex2(s[b][0] - m[b][0]), w01 = ex2(s[b][1] - m[b][1]), w10 = ex2(s[b][2] - m[b][0]), w11 = ex2(s[b][3] - m[b][1]);
            const uint32_t lo = ActF16::pack(w00, w01), hi = ActF16::pack(w10, w11);
            if (kTwice) {
                l[b][0] = fmaf(w00 + w10, back, l[b][0]);
                l[b][1] = fmaf(w01 + w11, back, l[b][1]);
                q0 = transpose8(ActF16::pack(w00 - ActF16::lo(lo), w01 - ActF16::hi(lo)));
                q1 = transpose8(ActF16::pack(w10 - ActF16::lo(hi), w11 - ActF16::hi(hi)));
            } else {
                l[b][0] = fmaf(kv8_total(w00, ActF16::lo(lo)) + kv8_total(w10, ActF16::lo(hi)), back, l[b][0]);
                l[b][1] = fmaf(kv8_total(w01, ActF16::hi(lo)) + kv8_total(w11, ActF16::hi(hi)), back, l[b][1]);
            }
            p0[b] = transpose8(lo);
            p1[b] = transpose8(hi);
        }
#pragma unroll
        for (int v = 0; v < kVVec; ++v) {
            uint32_t x[4][4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const uint4 u = *reinterpret_cast<const uint4*>(at + read_v + ((p & 1) + 8 * (p >> 1)) * HD + 128 * v);
                x[p][0] = u.x, x[p][1] = u.y, x[p][2] = u.z, x[p][3] = u.w;
            }
            if (key + kTile > most || isnan(ks)) {   // what no row of the tile attends; what stands in for a page that is not there
#pragma unroll
                for (int p = 0; p < 4; ++p)
                    if (key + 2 * t + (p & 1) + 8 * (p >> 1) >= most || isnan(ks)) x[p][0] = x[p][1] = x[p][2] = x[p][3] = 0u;
            }
#pragma unroll
            for (int d = 0; d < 8; ++d) {   // columns 2 d and 2 d + 1 of the lane's 16
                const uint32_t pick = d & 1 ? 0x7362u : 0x5140u;   // bytes 0, 1 or 2, 3 of two keys' words, key by key
                const uint32_t w0 = __byte_perm(x[0][d >> 1], x[1][d >> 1], pick), w1 = __byte_perm(x[2][d >> 1], x[3][d >> 1], pick);
                const uint32_t a0 = low_codes(w0), a1 = high_codes(w0), a2 = low_codes(w1), a3 = high_codes(w1);
#pragma unroll
                for (int b = 0; b < NT; ++b) mma_f16(o[b][8 * v + d], a0, a1, a2, a3, p0[b], p1[b]);
                if (kTwice) mma_f16(o[0][8 * v + d], a0, a1, a2, a3, q0, q1);
            }
        }
        const uint32_t next = stage == 0 ? S::kStages - 1 : stage - 1;   // (i + kStages - 1) % kStages
        if (i + S::kStages - 1 < mine) fetch(i + S::kStages - 1, next);
        asm volatile("cp.async.commit_group;" ::: "memory");
        stage = stage + 1 == S::kStages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");

    // the eight lanes of a pair add their totals; the warps' partial results meet in shared memory
    __syncthreads();   // the ring is free
    float* mine_at = reinterpret_cast<float*>(smem) + warp * (kPairs * S::kLd);
#pragma unroll
    for (int b = 0; b < NT; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float total = l[b][e];
            total += __shfl_xor_sync(0xffffffffu, total, 4);
            total += __shfl_xor_sync(0xffffffffu, total, 8);
            total += __shfl_xor_sync(0xffffffffu, total, 16);
            float* to = mine_at + (8 * b + 2 * t + e) * S::kLd;
            if (g == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(m[b][e], total);
#pragma unroll
            for (int v = 0; v < kVVec; ++v)
#pragma unroll
                for (int d = 0; d < 4; ++d)
                    *reinterpret_cast<float4*>(to + 128 * v + 16 * g + 4 * d) =
                        make_float4(o[b][8 * v + 2 * d][e], o[b][8 * v + 2 * d][2 + e], o[b][8 * v + 2 * d + 1][e], o[b][8 * v + 2 * d + 1][2 + e]);
        }
    __syncthreads();
    const float* all = reinterpret_cast<const float*>(smem);
    const bool whole = most <= a.chunk;   // this CTA has seen every key
    float* parts = a.part + static_cast<size_t>(tile_id) * a.chunks * (kPairs * S::kLd);
    const uint32_t here = min(kPairs, pairs - pair0);
    for (uint32_t e = threadIdx.x; e < here * (HD / 8); e += kThreads) {
        const uint32_t p = e / (HD / 8), d = e % (HD / 8) * 8;
        float top = kKv8None, total = 0.f, x[8] = {};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, all[(w * kPairs + p) * S::kLd + HD]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float* from = all + (w * kPairs + p) * S::kLd;
            const float by = ex2(from[HD] - top);
            total = fmaf(from[HD + 1], by, total);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(from[d + i], by, x[i]);
        }
        if (whole) {
            kv8_finish<Act>(a, r, pair0 + p, kvh, d, HD, total, x);
        } else {
            float* to = parts + (z * kPairs + p) * S::kLd;
            *reinterpret_cast<float4*>(to + d) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(to + d + 4) = make_float4(x[4], x[5], x[6], x[7]);
            if (d == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(top, total);
        }
    }
    if (whole) return;

    // The last of the tile's CTAs joins the chunks. Threads take 8 columns of a pair; where that leaves threads over they share the chunks
    // (`groups` of them, chunk k with group k % groups), and the groups' sums are added in order.
    const uint32_t chunks = (most + a.chunk - 1) / a.chunk;
    uint32_t* last = reinterpret_cast<uint32_t*>(smem + S::kSeen + 2 * kPairs * 4);
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) *last = atomicInc(a.done + tile_id, chunks - 1) == chunks - 1;   // the last arrival leaves 0
    __syncthreads();
    if (!*last) return;
    __threadfence();
    constexpr uint32_t kCols = HD / 8;
    const uint32_t items = here * kCols;
    const uint32_t groups = items >= kThreads ? 1u : kThreads / items, group = groups == 1 ? 0u : threadIdx.x / items;
    float* sums = reinterpret_cast<float*>(smem);   // [groups][here][kLd]
    for (uint32_t e = groups == 1 ? threadIdx.x : threadIdx.x % items; e < items && group < groups; e += kThreads) {
        const uint32_t p = e / kCols, d = e % kCols * 8;
        const float* from = parts + p * S::kLd;
        float top = kKv8None, total = 0.f, x[8] = {};
        for (uint32_t k0 = group; k0 < chunks; k0 += 4 * groups) {   // four chunks' loads in flight
            float2 ml[4];
            float4 u[4], w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t k = k0 + i * groups;
                const float* at = from + static_cast<size_t>(min(k, chunks - 1)) * (kPairs * S::kLd);
                ml[i] = __ldcg(reinterpret_cast<const float2*>(at + HD));
                u[i] = __ldcg(reinterpret_cast<const float4*>(at + d));
                w[i] = __ldcg(reinterpret_cast<const float4*>(at + d + 4));
                if (k >= chunks) ml[i] = make_float2(kKv8None, 0.f), u[i] = w[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            const float now = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), top), old = ex2(top - now);
            top = now;
            total *= old;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= old;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float by = ex2(ml[i].x - now), v[8] = {u[i].x, u[i].y, u[i].z, u[i].w, w[i].x, w[i].y, w[i].z, w[i].w};
                total = fmaf(ml[i].y, by, total);
#pragma unroll
                for (int c = 0; c < 8; ++c) x[c] = fmaf(v[c], by, x[c]);
            }
        }
        if (groups == 1) {
            kv8_finish<Act>(a, r, pair0 + p, kvh, d, HD, total, x);
        } else {
            float* to = sums + (group * here + p) * S::kLd;
            *reinterpret_cast<float4*>(to + d) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(to + d + 4) = make_float4(x[4], x[5], x[6], x[7]);
            if (d == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(top, total);
        }
    }
    if (groups == 1) return;
    __syncthreads();
    if (threadIdx.x < items) {
        const uint32_t p = threadIdx.x / kCols, d = threadIdx.x % kCols * 8;
        float top = kKv8None, total = 0.f, x[8] = {};
        for (uint32_t k = 0; k < groups; ++k) top = fmaxf(top, sums[(k * here + p) * S::kLd + HD]);
        for (uint32_t k = 0; k < groups; ++k) {
            const float* at = sums + (k * here + p) * S::kLd;
            const float by = ex2(at[HD] - top);
            total = fmaf(at[HD + 1], by, total);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fmaf(at[d + i], by, x[i]);
        }
        kv8_finish<Act>(a, r, pair0 + p, kvh, d, HD, total, x);
    }
}

typedef void (*attn_fn)(const Kv8Args);
struct Variant {
    attn_fn f;
    int bytes, threads, blocks;
};
template <typename Act>
Variant pick(uint32_t hd, uint32_t nt) {
#define DC_KV8_VARIANT(HD, NT) Variant{kv8_attn_kernel<Act, HD, NT>, static_cast<int>(Shape<HD, NT>::kBytes), Shape<HD, NT>::kThreads, Shape<HD, NT>::kBlocks}
    if (hd == 128) return nt == 1 ? DC_KV8_VARIANT(128, 1) : DC_KV8_VARIANT(128, 2);
    return nt == 1 ? DC_KV8_VARIANT(256, 1) : DC_KV8_VARIANT(256, 2);
#undef DC_KV8_VARIANT
}

// How a call is cut: tiles of 8 nt (row, head) pairs, chunks of `chunk` keys.
constexpr uint64_t kDoneCounters = DC_KV8_DONE_COUNTERS;
Kv8Cut cut_of(const dc_ctx* ctx, const dc_kv8_cache* c, uint32_t nq, uint32_t max_q, uint32_t max_len) {
    Kv8Cut t;
    // Pairs in eights, a CTA each: many narrow tiles hide their latencies better than few wide ones (24 pairs over 2,307 keys: 10.0 us in
    // eights, 12.1 in sixteens), until the tiles alone are more than the GPU holds at once; then two eights share a pass over the codes
    // (16 pairs of 64 x 1,200 keys: 44 against 52 us).
    const uint64_t eights = (static_cast<uint64_t>(max_q) * (nq / c->nkv) + 7) / 8;
    const uint32_t len = max_len;
    const uint64_t items = static_cast<uint64_t>(c->n_seqs) * c->nkv;
    Variant v = pick<dc::ActF16>(c->hd, 1);
    t.nt = eights > 1 && items * eights > static_cast<uint64_t>(ctx->sm_count) * v.blocks ? 2 : 1;
    v = pick<dc::ActF16>(c->hd, t.nt);
    t.tiles = static_cast<uint32_t>((eights + t.nt - 1) / t.nt);
    const uint64_t whole = items * t.tiles;
    const uint32_t warps = v.threads / 32, step = warps * kTile;   // a tile for each warp
    // Chunks. A join costs about 3 us and 0.1 us a chunk, a tile 0.5 us of its warp's time: keys of up to five tiles a warp stay whole
    // (603 keys of one request: 7.2 us whole, 7.7 cut in 10), others are cut in about sqrt(tiles of a warp * HD / 32), as long as every
    // SM has at most one set of eight warps to run (16,000 keys: 12.7 us in 18 chunks, 16.0 in 31; 131,071: 52.2 in 18, 54.4 in 37).
    uint64_t parts = 1;
    if (len > 5 * step && whole <= kDoneCounters) {
        const uint64_t room = static_cast<uint64_t>(ctx->sm_count) * 8 / warps / whole;
        parts = static_cast<uint64_t>(sqrt(static_cast<double>(len) / kTile * c->hd / 32 / warps));
        if (parts > room) parts = room < 1 ? 1 : room;
    }
    t.chunk = static_cast<uint32_t>(((len + parts - 1) / parts + step - 1) / step * step);
    t.chunks = (len + t.chunk - 1) / t.chunk;
    t.ctas = whole * t.chunks;
    t.part_bytes = t.chunks > 1 ? t.ctas * 8 * t.nt * (c->hd + 4) * sizeof(float) : 0;
    return t;
}

// The longest sequence that a call may meet.
uint32_t longest(const dc_kv8_cache* c, uint32_t max_len) {
    const uint32_t cap = c->max_pages * c->page_size;
    return max_len == 0 || max_len > cap ? cap : max_len;
}

// Whole tiles of the tensor cores (256 pairs a CTA, 128 of heads of 256) against eights: from 64 pairs a sequence and 2^29 products of a
// weight and a value on. Measured, us, tcgen05 and here, heads of 128: one sequence of 64 pairs (per kv head, of 8) over 2,307 keys 18.5 and 13.9,
// over 8,000 24.8 and 28.3; of 256 pairs over 600 keys 19.5 and 10.8, over 2,307 22.3 and 25.1; 16 sequences of 64 pairs over 1,000
// keys 28 and 36; 64 of 24 pairs over 1,200 keys 150 and 67. Heads of 256, 4 kv heads: 64 pairs over 8,000 keys 29.3 and 27.9; 16
// sequences of 64 pairs over 1,000 keys 29 and 48.
bool on_tcgen05(const dc_ctx* ctx, const dc_kv8_cache* c, uint32_t nq, uint32_t max_q, uint32_t max_len) {
    if (ctx->attn_engine != DC_ENGINE_TCGEN05) return false;
    const double pairs = static_cast<double>(max_q) * (nq / c->nkv);
    return pairs >= 64 && pairs * c->n_seqs * c->nkv * max_len * c->hd >= 536870912.0;
}

}  // namespace

int dc_kv8_attention_warm(dc_ctx* ctx) {
    static bool set[16] = {};
    if (set[ctx->device & 15]) return DC_OK;
    for (int i = 0; i < 8; ++i) {
        const uint32_t hd = i & 1 ? 256 : 128, nt = 1 + (i >> 1 & 1);
        const Variant v = i & 4 ? pick<dc::ActF16>(hd, nt) : pick<dc::ActBF16>(hd, nt);
        const cudaError_t e = cudaFuncSetAttribute(v.f, cudaFuncAttributeMaxDynamicSharedMemorySize, v.bytes);
        if (e != cudaSuccess) return dc_fail(ctx, DC_CUDA_ERROR, "kv8_attention: cannot opt in to %d bytes of shared memory: %s", v.bytes, cudaGetErrorString(e));
    }
    set[ctx->device & 15] = true;
    return DC_OK;
}

extern "C" size_t dc_kv8_attention_scratch_bytes(dc_ctx* ctx, const dc_kv8_cache* cache, uint32_t nq, uint32_t max_q, uint32_t max_len) {
    if (!ctx || dc_kv8_check(cache, nullptr, 0) != DC_OK || nq == 0 || nq % cache->nkv || max_q == 0) return 0;
    const uint32_t len = longest(cache, max_len);
    return (on_tcgen05(ctx, cache, nq, max_q, len) ? dc_kv8_attention_tc_cut(ctx, cache, nq, max_q, len) : cut_of(ctx, cache, nq, max_q, len)).part_bytes;
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
    if (static_cast<uint64_t>(max_q) * (nq / cache->nkv) >= (1ull << 28))
        return dc_fail(ctx, DC_UNSUPPORTED, "kv8_attention: max_q = %u rows of %u heads per kv head (below 2^28 together)", max_q, nq / cache->nkv);
    const dc_device_scope scope(ctx);
    const uint32_t len = longest(cache, max_len);
    const bool tc = on_tcgen05(ctx, cache, nq, max_q, len);
    const Kv8Cut t = tc ? dc_kv8_attention_tc_cut(ctx, cache, nq, max_q, len) : cut_of(ctx, cache, nq, max_q, len);   // as dc_kv8_attention_scratch_bytes says
    DC_REQUIRE(ctx, t.ctas < 0x7fffffffull, "kv8_attention: %llu CTAs: fewer rows or sequences a call", static_cast<unsigned long long>(t.ctas));
    Kv8Args a;
    a.c = *cache;
    a.c.k = static_cast<uint8_t*>(cache->k) + layer * cache->layer_stride;
    a.c.v = static_cast<uint8_t*>(cache->v) + layer * cache->layer_stride;
    a.c.k_scale = cache->k_scale + static_cast<size_t>(layer) * cache->n_pages * cache->nkv;
    a.c.v_scale = cache->v_scale + static_cast<size_t>(layer) * cache->n_pages * cache->nkv;
    a.part = nullptr;
    a.done = ctx->kv8_done;
    if (t.chunks > 1) {
        void* ws = nullptr;
        if ((rc = dc_stream_workspace(ctx, static_cast<cudaStream_t>(stream), t.part_bytes, "kv8_attention", &ws)) != DC_OK) return rc;
        a.part = static_cast<float*>(ws);
    }
    if ((rc = dc_kv8_attention_warm(ctx)) != DC_OK) return rc;
    a.q = static_cast<const uint16_t*>(q);
    a.gate = gate;
    a.q_start = q_start;
    a.qpos = qpos;
    a.y = static_cast<uint16_t*>(y);
    a.status = ctx->status_dev;
    a.rows = rows, a.ldq = ldq, a.ldg = ldg, a.ldy = ldy, a.group = nq / cache->nkv, a.max_q = max_q, a.max_len = len;
    a.tiles = t.tiles, a.chunk = t.chunk, a.chunks = t.chunks;
    a.page_shift = __builtin_ctz(cache->page_size), a.group_inverse = a.group > 1 ? static_cast<uint32_t>((1ull << 32) / a.group + 1) : 0u;
    a.scale = kKv8Log2e / sqrtf(static_cast<float>(cache->hd));
    const bool f16 = ctx->act_dtype == DC_ACT_F16;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (tc) return dc_kv8_attention_tc(ctx, s, a, t.ctas);
    const Variant v = f16 ? pick<dc::ActF16>(cache->hd, t.nt) : pick<dc::ActBF16>(cache->hd, t.nt);
    return dc_kv8_launch(ctx, "kv8_attention", v.f, 2 * t.ctas <= static_cast<uint64_t>(ctx->sm_count), dim3(static_cast<uint32_t>(t.ctas)), v.threads, v.bytes, s, a);
}
