// What the two kernels of dc_kv8_attention share: the arguments of a launch, the rows of a tile, conversions, the end of a row.
#pragma once
#include "kv8.cuh"

namespace dc {

constexpr float kKv8None = -1e30f;   // running maximum of a row that has seen nothing
// Weights are 2^(t - m) in fp16, t a term's exponent. m is set to 2^7 below the largest term and follows it when that has grown by 2^8 more, so
// that the largest weight is between 2^7 and 2^15: fp16's upper end. Its 11 bits then reach down to 2^-21 of the row's largest term and its last one to
// 2^-31 (with m at the largest term itself, 2^-14 and 2^-24: beside a key of 2^26 times the weight all others were lost).
constexpr float kKv8Below = 7.0f;
constexpr float kKv8Step = kKv8Below + 8.0f;
constexpr float kKv8Log2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The two codes in the low (high) 16 bits as fp16, exactly.
__device__ __forceinline__ uint32_t low_codes(uint32_t w) {
    uint32_t h;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(h) : "r"(w));
    return h;
}
__device__ __forceinline__ uint32_t high_codes(uint32_t w) {
    uint32_t h;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(h) : "r"(w));
    return h;
}

// The rows of a tile: what the kernel and the join agree on.
struct Kv8Rows {
    uint32_t start, count, len;   // of the sequence: first packed row, rows, tokens
    bool ok;
};
__device__ __forceinline__ Kv8Rows kv8_rows(const dc_kv8_cache& c, const uint32_t* q_start, uint32_t j, uint32_t rows, uint32_t max_q) {
    Kv8Rows r;
    r.start = q_start[j];
    const uint32_t end = q_start[j + 1];
    r.len = c.lens[j];
    r.count = end - r.start;
    r.ok = end >= r.start && end <= rows && r.count <= max_q;
    return r;
}
// Tokens that row i of the sequence attends; *past is set where its position lies at or past the length.
__device__ __forceinline__ uint32_t kv8_visible(const Kv8Rows& r, const uint32_t* qpos, uint32_t i, bool* past) {
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

struct Kv8Args {
    dc_kv8_cache c;   // k, v and the scales point at the layer
    const uint16_t* q;
    const float* gate;
    const uint32_t* q_start;
    const uint32_t* qpos;
    uint16_t* y;
    float* part;
    uint32_t* done;   // a counter per tile, zero between launches
    int* status;
    uint32_t rows, ldq, ldg, ldy, group, max_q, max_len, tiles, chunk, chunks, page_shift, group_inverse;
    float scale;      // hd^-1/2 log2(e)
};

// pair / group: pairs are below 2^28 and groups at most 16, so the product with floor(2^32 / group) + 1 is exact.
__device__ __forceinline__ uint32_t kv8_row_of(const Kv8Args& a, uint32_t pair) { return a.group == 1 ? pair : __umulhi(pair, a.group_inverse); }

// The largest magnitude of a query row, as 16 bits; WORDS 8-byte pieces a lane holds of it, `lanes` (16 or 32) lanes hold the row.
template <int WORDS>
__device__ __forceinline__ uint32_t kv8_query_top(const uint2* x, int lanes = 32) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < WORDS; ++i) top = __vmaxu2(top, __vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu));
    top = max(top & 0xffffu, top >> 16);
    if (lanes == 32) return __reduce_max_sync(0xffffffffu, top);
#pragma unroll
    for (int o = 8; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    return top;
}
// A bf16 row is divided by a power of two that brings its largest magnitude to [2^14, 2^15): then its 8 bits fit fp16 but for elements
// 2^-28 below it. fp16 rows stay as they are. Returns the divisor; NaN for a row that is not finite.
template <typename Act, int WORDS>
__device__ __forceinline__ float kv8_query_row(uint2* x, uint32_t top) {
    float up = 1.f;
    if (Act::kUmmaFormat == 1) {
        const uint32_t e = top >> 7;   // exponent field of the largest
        // 2^(e - 127) -> 2^14; fields beyond 1 .. 254 (zeros, subnormals, infinities) take the nearest
        const int shift = min(max(static_cast<int>(e), 1), 254) - 127 - 14;
        const int half = shift / 2;   // two factors: 2^-shift alone may pass fp32's exponents
        const float down = kv8_exp2i(-half), rest_down = kv8_exp2i(-(shift - half));
#pragma unroll
        for (int i = 0; i < WORDS; ++i) {
            x[i].x = ActF16::pack(Act::lo(x[i].x) * down * rest_down, Act::hi(x[i].x) * down * rest_down);
            x[i].y = ActF16::pack(Act::lo(x[i].y) * down * rest_down, Act::hi(x[i].y) * down * rest_down);
        }
        up = kv8_exp2i(half) * kv8_exp2i(shift - half);
    }
    return Act::one(static_cast<uint16_t>(top)) <= 3.4028235e38f ? up : __uint_as_float(0x7fffffffu);
}

// The gate of columns d .. d + 7 of a pair.
__device__ __forceinline__ void kv8_gate8(const Kv8Args& a, const Kv8Rows& r, uint32_t pair, uint32_t kvh, uint32_t d, uint32_t hd, float4 (&g)[2]) {
    const uint32_t of = kv8_row_of(a, pair);
    const float4* from = reinterpret_cast<const float4*>(a.gate + static_cast<size_t>(r.start + of) * a.ldg + (kvh * a.group + pair - of * a.group) * hd + d);
    g[0] = from[0];
    g[1] = from[1];
}
// (reciprocal and exponential to 2^-21: the output has at most 11 bits)
__device__ __forceinline__ float kv8_sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }
// Eight finished columns of a pair: gate (where there is one), 16 bits.
template <typename Act>
__device__ __forceinline__ void kv8_store8(const Kv8Args& a, const Kv8Rows& r, uint32_t pair, uint32_t kvh, uint32_t d, uint32_t hd, float4 x, float4 y, const float4 (&g)[2]) {
    const uint32_t of = kv8_row_of(a, pair);
    if (a.gate) {
        x = make_float4(x.x * kv8_sigmoid(g[0].x), x.y * kv8_sigmoid(g[0].y), x.z * kv8_sigmoid(g[0].z), x.w * kv8_sigmoid(g[0].w));
        y = make_float4(y.x * kv8_sigmoid(g[1].x), y.y * kv8_sigmoid(g[1].y), y.z * kv8_sigmoid(g[1].z), y.w * kv8_sigmoid(g[1].w));
    }
    *reinterpret_cast<uint4*>(a.y + static_cast<size_t>(r.start + of) * a.ldy + (kvh * a.group + pair - of * a.group) * hd + d) =
        make_uint4(Act::pack(x.x, x.y), Act::pack(x.z, x.w), Act::pack(y.x, y.y), Act::pack(y.z, y.w));
}

// Columns d .. d + 7 of a pair: sums over the total, then as above. A row that attends nothing has no total: zero.
template <typename Act>
__device__ __forceinline__ void kv8_finish(const Kv8Args& a, const Kv8Rows& r, uint32_t pair, uint32_t kvh, uint32_t d, uint32_t hd, float total, float (&o)[8]) {
    const float by = total == 0.f ? 0.f : 1.0f / total;
    float4 g[2];
    if (a.gate) kv8_gate8(a, r, pair, kvh, d, hd, g);
    kv8_store8<Act>(a, r, pair, kvh, d, hd, make_float4(o[0] * by, o[1] * by, o[2] * by, o[3] * by), make_float4(o[4] * by, o[5] * by, o[6] * by, o[7] * by), g);
}

}  // namespace dc

// How a call is cut: tiles of (row, head) pairs (8 nt each in kv8_attn.cu), chunks of keys, the CTAs and the scratch that makes.
struct Kv8Cut {
    uint32_t nt = 0, tiles = 0, chunk = 0, chunks = 0;
    uint64_t ctas = 0, part_bytes = 0;
};
// The tcgen05 form (kv8_attn_tc.cu).
Kv8Cut dc_kv8_attention_tc_cut(const dc_ctx* ctx, const dc_kv8_cache* c, uint32_t nq, uint32_t max_q, uint32_t max_len);
int dc_kv8_attention_tc(dc_ctx* ctx, cudaStream_t s, const dc::Kv8Args& a, uint64_t ctas);
