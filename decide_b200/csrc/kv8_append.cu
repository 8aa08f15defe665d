// dc_kv8_append: new K and V rows of one layer into the pages of the 8-bit cache.
//
// For a (page, kv head): amax over the new rows, e = the least exponent with 448 * 2^e >= amax, scale = 2^e (a page that already
// holds tokens: the larger of that and its scale), code = e4m3(x / scale). The division is a multiplication by a power of two, so
// every code is one exact rounding of the 16-bit input. When the scale of a page that holds tokens rises, their codes are
// rounded again at the new one.
//
// Bound by memory: 2 bytes in and 1 byte out a value. One CTA per (page that the call touches, kv head): the new rows of a page, K and V,
// fit the CTA's registers (at most 128 tokens x 256 values x 2 over 256 threads), so the rows are read once, and before the page is
// known: their place depends on the offsets and the length alone. amax is taken on the packed 16-bit magnitudes (an integer maximum:
// the order of the bit patterns is that of the magnitudes, infinities and NaN above all finite ones), one block reduction for K and V
// together, then the conversion. CTAs share nothing, so no order of execution changes a result.
// Measured on the device: 64 x 603 rows, 8 heads of 128, 43.9 us (237 MB, 5.4 TB/s; 56 us with K and V in CTAs of their own that looked the
// page up first); a token for each of 64 sequences 3.2 us.
#include "kv8.cuh"

namespace {

using namespace dc;

constexpr int kThreads = 256;

// What K or V does with its new rows once their largest magnitude is known: the page's scale, the codes that are there again if it rose, the new codes.
template <typename Act, int VECS>
__device__ __forceinline__ void write_rows(const dc_kv8_cache& c, uint8_t* dst, float* scale_at, float before, uint32_t offset, uint32_t vectors,
                                           uint32_t row_shift, uint32_t top, const uint4 (&x)[VECS]) {
    const float amax = Act::one(static_cast<uint16_t>(top));
    float scale = kv8_exp2i(kv8_exponent(amax));
    if (offset) scale = isnan(before) ? before : fmaxf(before, scale);
    if (!(amax <= 3.4028235e38f)) scale = __uint_as_float(0x7fffffffu);   // a value that is not finite: NaN
    const bool poisoned = isnan(scale);
    const float inverse = poisoned ? 0.f : 1.0f / scale;
    if (offset && scale > before) {   // tokens 0 .. offset of the page at the new scale
        const float ratio = before * inverse;
        for (uint32_t e = threadIdx.x; e < offset << (row_shift - 1); e += kThreads) {
            uint4* at = reinterpret_cast<uint4*>(dst + static_cast<size_t>(e >> (row_shift - 1)) * c.token_stride + 16 * (e & ((1u << (row_shift - 1)) - 1)));
            uint4 w = *at;
            uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = e4m3x2_to_float2(static_cast<uint16_t>(u[i])), b = e4m3x2_to_float2(static_cast<uint16_t>(u[i] >> 16));
                u[i] = e4m3x2(a.x * ratio, a.y * ratio) | (static_cast<uint32_t>(e4m3x2(b.x * ratio, b.y * ratio)) << 16);
            }
            *at = w;
        }
    }
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const uint32_t e = threadIdx.x + i * kThreads;
        if (e >= vectors) break;
        const uint32_t in[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        uint32_t out[2] = {0u, 0u};
        if (!poisoned) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                out[h] = e4m3x2(Act::lo(in[2 * h]) * inverse, Act::hi(in[2 * h]) * inverse) |
                         (static_cast<uint32_t>(e4m3x2(Act::lo(in[2 * h + 1]) * inverse, Act::hi(in[2 * h + 1]) * inverse)) << 16);
        }
        *reinterpret_cast<uint2*>(dst + static_cast<size_t>(offset + (e >> row_shift)) * c.token_stride + 8 * (e & ((1u << row_shift) - 1))) = make_uint2(out[0], out[1]);
    }
    if (threadIdx.x == 0) *scale_at = scale;
}

// VECS: 16-byte vectors (8 values) a thread holds of a page's new rows, of K and of V.
template <typename Act, int VECS>
__global__ void __launch_bounds__(kThreads)
kv8_append_kernel(dc_kv8_cache c, uint32_t page_shift, uint32_t row_shift, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, uint32_t ldk,
                  uint32_t ldv, const uint32_t* __restrict__ row_start, uint32_t rows, uint32_t max_rows, int* __restrict__ status) {
    kv8_begin();
    const uint32_t j = blockIdx.z, head = blockIdx.y;
    const bool reports = head == 0 && threadIdx.x == 0;
    const uint32_t r0 = row_start[j], r1 = row_start[j + 1], len = c.lens[j];
    if (r1 == r0) return;
    if (r1 < r0 || r1 > rows || r1 - r0 > max_rows || r1 - r0 > len) {
        if (reports) kv8_flag(status, DC_STATUS_KV8_OFFSETS);
        return;
    }
    if (len > c.max_pages << page_shift) {
        if (reports) kv8_flag(status, DC_STATUS_KV8_LENGTH);
        return;
    }
    const uint32_t begin = len - (r1 - r0);                        // position of row r0
    const uint32_t column = (begin >> page_shift) + blockIdx.x;    // column of the table
    const uint32_t first = column << page_shift;                   // position of the page's first token
    if (first >= len) return;
    const uint32_t page = c.table[static_cast<size_t>(j) * c.max_pages + column];
    const uint32_t lo = max(begin, first), hi = min(len, first + c.page_size);
    const uint32_t offset = lo - first, vectors = (hi - lo) << row_shift;   // the new rows' place in the page
    const size_t from = r0 + lo - begin, col = static_cast<size_t>(head) * c.hd;

    uint4 kx[VECS], vx[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        const uint32_t e = threadIdx.x + i * kThreads;
        const size_t row = from + (e >> row_shift), at = col + 8 * (e & ((1u << row_shift) - 1));
        kx[i] = vx[i] = make_uint4(0, 0, 0, 0);
        if (e < vectors) {
            kx[i] = __ldg(reinterpret_cast<const uint4*>(k + row * ldk + at));
            vx[i] = __ldg(reinterpret_cast<const uint4*>(v + row * ldv + at));
        }
    }
    if (page >= c.n_pages) {
        if (reports) kv8_flag(status, DC_STATUS_KV8_PAGE);
        return;
    }
    const uint32_t holders = c.refs[page];
    const size_t scale_at = static_cast<size_t>(page) * c.nkv + head;
    const float k_before = offset ? c.k_scale[scale_at] : 0.f, v_before = offset ? c.v_scale[scale_at] : 0.f;

    uint32_t k_top = 0, v_top = 0;   // two 16-bit magnitudes each
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
        k_top = __vmaxu2(__vmaxu2(k_top, __vmaxu2(kx[i].x & 0x7fff7fffu, kx[i].y & 0x7fff7fffu)), __vmaxu2(kx[i].z & 0x7fff7fffu, kx[i].w & 0x7fff7fffu));
        v_top = __vmaxu2(__vmaxu2(v_top, __vmaxu2(vx[i].x & 0x7fff7fffu, vx[i].y & 0x7fff7fffu)), __vmaxu2(vx[i].z & 0x7fff7fffu, vx[i].w & 0x7fff7fffu));
    }
    k_top = __reduce_max_sync(0xffffffffu, max(k_top & 0xffffu, k_top >> 16));
    v_top = __reduce_max_sync(0xffffffffu, max(v_top & 0xffffu, v_top >> 16));
    __shared__ uint2 tops[kThreads / 32];
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = make_uint2(k_top, v_top);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        k_top = max(k_top, tops[w].x);
        v_top = max(v_top, tops[w].y);
    }
    if (holders != 1u) {
        if (reports) kv8_flag(status, DC_STATUS_KV8_SHARED);
        return;
    }
    const uint64_t page_at = page * c.page_stride + head * c.head_stride;
    write_rows<Act, VECS>(c, static_cast<uint8_t*>(c.k) + page_at, c.k_scale + scale_at, k_before, offset, vectors, row_shift, k_top, kx);
    write_rows<Act, VECS>(c, static_cast<uint8_t*>(c.v) + page_at, c.v_scale + scale_at, v_before, offset, vectors, row_shift, v_top, vx);
}

template <typename Act>
int launch(dc_ctx* ctx, dim3 grid, cudaStream_t s, uint32_t vecs, const dc_kv8_cache& c, const uint16_t* k, const uint16_t* v, uint32_t ldk, uint32_t ldv,
            const uint32_t* row_start, uint32_t rows, uint32_t max_rows) {
    auto kern = vecs <= 1 ? kv8_append_kernel<Act, 1> : vecs <= 2 ? kv8_append_kernel<Act, 2> : vecs <= 4 ? kv8_append_kernel<Act, 4>
              : vecs <= 8 ? kv8_append_kernel<Act, 8> : kv8_append_kernel<Act, 16>;
    return dc_kv8_launch(ctx, "kv8_append", kern, false, grid, kThreads, 0, s, c, __builtin_ctz(c.page_size), __builtin_ctz(c.hd / 8), k, v, ldk, ldv, row_start, rows,
                         max_rows, ctx->status_dev);
}

}  // namespace

extern "C" int dc_kv8_append(dc_ctx* ctx, void* stream, const dc_kv8_cache* cache, uint32_t layer, const void* k, const void* v, uint32_t ldk,
                             uint32_t ldv, const uint32_t* row_start, uint32_t rows, uint32_t max_rows) {
    if (!ctx) return DC_INVALID_ARG;
    int rc = dc_kv8_require(ctx, "kv8_append", cache);
    if (rc != DC_OK) return rc;
    DC_REQUIRE(ctx, k && v && row_start, "kv8_append: null operand");
    DC_REQUIRE(ctx, layer < cache->layers, "kv8_append: layer %u of %u", layer, cache->layers);
    const uint64_t width = static_cast<uint64_t>(cache->nkv) * cache->hd;
    DC_REQUIRE(ctx, ldk >= width && ldv >= width && ldk % 8 == 0 && ldv % 8 == 0,
               "kv8_append: ldk = %u, ldv = %u must cover nkv * hd = %llu and be multiples of 8", ldk, ldv, static_cast<unsigned long long>(width));
    DC_REQUIRE(ctx, reinterpret_cast<uintptr_t>(k) % 16 == 0 && reinterpret_cast<uintptr_t>(v) % 16 == 0, "kv8_append: k and v must be 16-byte aligned");
    if (rows == 0 || max_rows == 0) return DC_OK;   // no rows: nothing to write
    const dc_device_scope scope(ctx);
    dc_kv8_cache c = *cache;
    c.k = static_cast<uint8_t*>(c.k) + layer * c.layer_stride;
    c.v = static_cast<uint8_t*>(c.v) + layer * c.layer_stride;
    c.k_scale += static_cast<size_t>(layer) * c.n_pages * c.nkv;
    c.v_scale += static_cast<size_t>(layer) * c.n_pages * c.nkv;
    const uint32_t most = max_rows < rows ? max_rows : rows;
    // most rows touch at most this many pages: the first of them may be in the middle of a page
    const uint32_t spans = most / c.page_size + (most % c.page_size > 1 ? 2u : 1u);
    const uint32_t fit = most < c.page_size ? most : c.page_size;
    const uint32_t vecs = (fit * (c.hd / 8) + kThreads - 1) / kThreads;
    auto go = ctx->act_dtype == DC_ACT_F16 ? launch<dc::ActF16> : launch<dc::ActBF16>;
    return go(ctx, dim3(spans, c.nkv, c.n_seqs), static_cast<cudaStream_t>(stream), vecs, c, static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v),
              ldk, ldv, row_start, rows, max_rows);
}
