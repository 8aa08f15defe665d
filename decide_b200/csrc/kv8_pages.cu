// Page bookkeeping of the paged 8-bit K/V cache: dc_kv8_extend, dc_kv8_fork, dc_kv8_free, dc_kv8_compact.
//
// Integers and copies. Which page goes where is decided on the device, so that a serving loop never waits for the host and the
// calls can be captured: one CTA validates the request, decides (a page is free when refs is 0; the i-th page needed is the i-th
// free one, found by block scans over refs) and writes table, refs and lens; where pages move, it leaves a list of (from, to) in
// the workspace for a second kernel that copies them in every layer with the whole GPU. Nothing depends on the order in which
// threads run: counts are integer atomics, places come from scans.
//
// What bounds them: the deciding CTA is a chain of a few block-wide steps (latency; refs are read 16 bytes a thread), the copying
// kernel is bound by memory (a page-head block of page_size * hd codes, contiguous in the default layout, per warp step).
// Measured on the device: copies of four states of 2,307 tokens in nine layers 62 us (350 MB, 5.7 TB/s with
// the deciding kernel); eight forks that share, grow, half of them freed, the cache closed up: 24 us in six kernels (27.6 with the forks'
// sequences and lengths loaded again by each step, and rows split by divisions in the copying kernel).
#include "kv8.cuh"

namespace {

using namespace dc;

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;

// Workspace of a call: a header, then per page the moves (from, to) and one word (the free pages found, or where a page moved).
struct Plan {
    uint32_t* head;   // [0] moves
    uint2* moves;     // [n_pages]
    uint32_t* slots;  // [n_pages]
};
__host__ __device__ inline size_t plan_bytes(uint32_t n_pages) { return 64 + static_cast<size_t>(n_pages) * 12; }
__host__ __device__ inline Plan plan_at(void* ws, uint32_t n_pages) {
    Plan p;
    p.head = static_cast<uint32_t*>(ws);
    p.moves = reinterpret_cast<uint2*>(p.head + 16);
    p.slots = reinterpret_cast<uint32_t*>(p.moves + n_pages);
    return p;
}

// Exclusive prefix sum over the block's threads; *total gets the sum of all. One barrier: every warp adds up the warps' sums for itself.
// `sums`: 2 x 32 words of shared memory, used in turn (`turn` counts the calls), so that a call does not wait for the last one's readers.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* sums, uint32_t& turn, uint32_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t s = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += y;
    }
    uint32_t* mine = sums + 32 * (turn++ & 1u);
    if (lane == 31) mine[warp] = s;
    __syncthreads();
    uint32_t t = mine[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, t, o);
        if (lane >= o) t += y;
    }
    *total = __shfl_sync(0xffffffffu, t, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, t, max(warp - 1, 0));
    return (warp ? before : 0u) + s - x;
}

// The first `need` pages with refs 0, ascending, into slots; returns how many there are, at most `need`. The caller's writes to refs
// are behind a barrier.
__device__ uint32_t find_free(const uint32_t* refs, uint32_t n_pages, uint32_t need, uint32_t* slots, uint32_t* sums, uint32_t& turn) {
    uint32_t found = 0;
    for (uint32_t base = 0; base < n_pages && found < need; base += 4 * kPlanThreads) {
        const uint32_t at = base + 4 * threadIdx.x;
        uint32_t mask = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < n_pages && __ldcg(refs + at + i) == 0u) mask |= 1u << i;
        uint32_t total;
        uint32_t place = found + block_scan(__popc(mask), sums, turn, &total);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (mask >> i & 1u) {
                if (place < need) slots[place] = at + i;
                ++place;
            }
        found += total;
    }
    return min(found, need);
}

// A sequence's pages, from its length as it is now; flags a length that its row of the table cannot hold.
__device__ __forceinline__ bool length_fits(const dc_kv8_cache& c, uint32_t len) { return len <= c.max_pages * c.page_size; }

// refs of the pages of sequence j of `len` tokens, by one warp: `by` = -1 gives them up, + 1 takes them back, 0 only looks at the table. *bad is
// set where a page id is outside the pool (it is passed over) or a page that nobody held is given up.
__device__ __forceinline__ void hold(const dc_kv8_cache& c, uint32_t j, uint32_t len, int by, int* bad) {
    const uint32_t pages = kv8_pages(len, c.page_size);
    for (uint32_t col = threadIdx.x & 31; col < pages; col += 32) {
        const uint32_t page = c.table[static_cast<size_t>(j) * c.max_pages + col];
        if (page >= c.n_pages) *bad = DC_STATUS_KV8_PAGE;
        else if (by != 0 && atomicAdd(&c.refs[page], static_cast<uint32_t>(by)) == 0u && by < 0) *bad = DC_STATUS_KV8_REFS;
    }
}

__global__ void __launch_bounds__(kPlanThreads)
extend_kernel(dc_kv8_cache c, const uint32_t* add, Plan plan, int* status) {
    __shared__ uint32_t sums[64], few[kPlanThreads];
    __shared__ int bad;
    uint32_t turn = 0;
    kv8_begin();
    if (threadIdx.x == 0) bad = 0;
    __syncthreads();
    // what each sequence lacks, and how many pages the ones before it in the round lack
    uint32_t need = 0, held = 0, mine = 0, len = 0, more = 0, place = 0;
    auto look = [&](uint32_t base, uint32_t* total) {
        const uint32_t j = base + threadIdx.x;
        held = mine = len = more = 0;
        if (j < c.n_seqs) {
            len = c.lens[j];
            more = add[j];
            const uint64_t after = static_cast<uint64_t>(len) + more;
            if (after > static_cast<uint64_t>(c.max_pages) * c.page_size) {
                bad = DC_STATUS_KV8_LENGTH;
            } else {
                held = kv8_pages(len, c.page_size);
                mine = kv8_pages(static_cast<uint32_t>(after), c.page_size) - held;
            }
        }
        // 1024 of at most 2^21 + 1 each: fits 32 bits
        return block_scan(min(mine, c.n_pages + 1), sums, turn, total);
    };
    for (uint32_t base = 0; base < c.n_seqs; base += kPlanThreads) {
        uint32_t total;
        place = look(base, &total);
        need = min(need + total, c.n_pages + 1);   // more than the pool is too many, however many
    }
    __syncthreads();
    uint32_t* slots = need <= kPlanThreads ? few : plan.slots;
    if (bad || need > c.n_pages || find_free(c.refs, c.n_pages, need, slots, sums, turn) < need) {
        if (threadIdx.x == 0) kv8_flag(status, bad ? bad : DC_STATUS_KV8_POOL);
        return;
    }
    __syncthreads();
    uint32_t given = 0;
    for (uint32_t base = 0; base < c.n_seqs; base += kPlanThreads) {
        if (c.n_seqs > kPlanThreads) {   // otherwise the one round above still stands
            uint32_t total;
            place = given + look(base, &total);
            given += total;
        }
        const uint32_t j = base + threadIdx.x;
        for (uint32_t i = 0; i < mine; ++i) {
            const uint32_t page = slots[place + i];
            c.table[static_cast<size_t>(j) * c.max_pages + held + i] = page;
            c.refs[page] = 1u;
        }
        if (j < c.n_seqs) c.lens[j] = len + more;
    }
}

// Pages that fork i copies (the rest of its source's pages it shares).
__device__ __forceinline__ uint32_t copied_pages(const dc_kv8_cache& c, uint32_t len, bool deep) {
    return deep ? kv8_pages(len, c.page_size) : (len % c.page_size != 0u ? 1u : 0u);
}

__global__ void __launch_bounds__(kPlanThreads)
fork_kernel(dc_kv8_cache c, const uint32_t* src, const uint32_t* dst, uint32_t n, bool deep, Plan plan, int* status) {
    extern __shared__ uint32_t taken[];   // one bit a sequence: it is a destination
    __shared__ uint32_t sums[64], few[kPlanThreads], places[kPlanThreads];
    __shared__ uint4 named[kPlanThreads];   // of up to 1024 forks: source, destination, their lengths (each step would load them again otherwise)
    __shared__ int bad;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const bool one_round = n <= kPlanThreads;
    uint32_t turn = 0;
    kv8_begin();
    for (uint32_t i = threadIdx.x; i < (c.n_seqs + 31) / 32; i += kPlanThreads) taken[i] = 0u;
    if (threadIdx.x == 0) {
        bad = 0;
        plan.head[0] = 0u;
    }
    __syncthreads();
    // what the forks name, and how many pages they copy: `place` of them before this thread's in the round
    uint32_t need = 0, place = 0;
    for (uint32_t base = 0; base < n; base += kPlanThreads) {
        const uint32_t i = base + threadIdx.x;
        uint32_t copied = 0, total;
        if (i < n) {
            const uint32_t d = dst[i], s = src[i];
            if (d >= c.n_seqs || s >= c.n_seqs) {
                bad = DC_STATUS_KV8_SEQUENCE;
            } else {
                const uint32_t d_len = c.lens[d], s_len = c.lens[s];
                if (atomicOr(&taken[d >> 5], 1u << (d & 31)) >> (d & 31) & 1u) bad = DC_STATUS_KV8_SEQUENCE;
                if (!length_fits(c, d_len) || !length_fits(c, s_len)) bad = DC_STATUS_KV8_LENGTH;
                else copied = min(copied_pages(c, s_len, deep), c.n_pages + 1);
                named[threadIdx.x] = make_uint4(s, d, s_len, d_len);
            }
        }
        place = block_scan(copied, sums, turn, &total);
        places[threadIdx.x] = place;   // read as they are where there is one round
        need = min(need + total, c.n_pages + 1);
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n && !bad; i += kPlanThreads) {
        const uint32_t s = one_round ? named[i].x : src[i];
        if (taken[s >> 5] >> (s & 31) & 1u) bad = DC_STATUS_KV8_SEQUENCE;
    }
    __syncthreads();
    if (bad) {
        if (threadIdx.x == 0) kv8_flag(status, bad);
        return;
    }
    auto fork_at = [&](uint32_t i) {   // as named[i], past the first 1024 too
        if (one_round) return named[i];
        const uint32_t s = src[i], d = dst[i];
        return make_uint4(s, d, c.lens[s], c.lens[d]);
    };
    // the destinations give up what they hold; what the sources hold has to name pages
    for (uint32_t i = warp; i < 2 * n; i += kPlanThreads / 32) {
        const uint4 f = fork_at(i >> 1);
        if (i & 1u) hold(c, f.y, f.w, -1, &bad);
        else hold(c, f.x, f.z, 0, &bad);
    }
    __syncthreads();
    uint32_t* slots = need <= kPlanThreads ? few : plan.slots;
    const bool enough = !bad && need <= c.n_pages && find_free(c.refs, c.n_pages, need, slots, sums, turn) == need;
    __syncthreads();
    if (!enough) {   // as it was
        const int what = bad ? bad : DC_STATUS_KV8_POOL;
        __syncthreads();
        for (uint32_t i = warp; i < n; i += kPlanThreads / 32) {
            const uint4 f = fork_at(i);
            hold(c, f.y, f.w, 1, &bad);
        }
        if (threadIdx.x == 0) kv8_flag(status, what);
        return;
    }
    uint32_t given = 0;
    for (uint32_t base = 0; base < n; base += kPlanThreads) {
        if (!one_round) {
            const uint32_t i = base + threadIdx.x;
            uint32_t total;
            place = given + block_scan(i < n ? copied_pages(c, fork_at(i).z, deep) : 0u, sums, turn, &total);
            given += total;
            __syncthreads();
            places[threadIdx.x] = place;
            __syncthreads();
        }
        // warps over the round's forks, lanes over the pages; a fork's place comes from the warp that scanned it
        for (uint32_t k = warp; k < kPlanThreads && base + k < n; k += kPlanThreads / 32) {
            const uint4 f = fork_at(base + k);
            const uint32_t pages = kv8_pages(f.z, c.page_size), copied = copied_pages(c, f.z, deep), shared = pages - copied;
            const uint32_t* from = c.table + static_cast<size_t>(f.x) * c.max_pages;
            uint32_t* to = c.table + static_cast<size_t>(f.y) * c.max_pages;
            for (uint32_t col = lane; col < pages; col += 32) {
                uint32_t page = from[col];
                if (col < shared) {
                    atomicAdd(&c.refs[page], 1u);
                } else {
                    const uint32_t slot = places[k] + col - shared, fresh = slots[slot];
                    plan.moves[slot] = make_uint2(page, fresh);
                    c.refs[fresh] = 1u;
                    page = fresh;
                }
                to[col] = page;
            }
        }
    }
    __syncthreads();   // `lens` are read above where there are several rounds
    for (uint32_t i = threadIdx.x; i < n; i += kPlanThreads) {
        if (one_round) c.lens[named[i].y] = named[i].z;
        else c.lens[dst[i]] = c.lens[src[i]];
    }
    if (threadIdx.x == 0) plan.head[0] = need;
}

__global__ void __launch_bounds__(128) free_kernel(dc_kv8_cache c, const uint32_t* seqs, int* status) {
    kv8_begin();
    const uint32_t j = seqs[blockIdx.x];
    __shared__ uint32_t claimed;
    if (threadIdx.x == 0) {
        claimed = 0u;
        if (j >= c.n_seqs) kv8_flag(status, DC_STATUS_KV8_SEQUENCE);
        else if (!length_fits(c, c.lens[j])) kv8_flag(status, DC_STATUS_KV8_LENGTH);
        else claimed = atomicExch(&c.lens[j], 0u);   // whoever comes second finds an empty sequence
    }
    __syncthreads();
    const uint32_t pages = kv8_pages(claimed, c.page_size);
    for (uint32_t col = threadIdx.x; col < pages; col += 128) {
        const uint32_t page = c.table[static_cast<size_t>(j) * c.max_pages + col];
        if (page >= c.n_pages) {
            kv8_flag(status, DC_STATUS_KV8_PAGE);
            continue;
        }
        // Several sequences of the call may name a page that fewer hold. Whoever finds none left, or fewer than none while another is about to put
        // its own back, puts it back: none does so before all that were held are gone, so the count ends at zero.
        if (static_cast<int>(atomicSub(&c.refs[page], 1u)) <= 0) {
            atomicAdd(&c.refs[page], 1u);
            kv8_flag(status, DC_STATUS_KV8_REFS);
        }
    }
}

__global__ void __launch_bounds__(kPlanThreads) compact_kernel(dc_kv8_cache c, Plan plan, uint32_t* live_out) {
    __shared__ uint32_t sums[64];
    uint32_t turn = 0, live = 0, mask = 0;   // of four pages, those in use
    kv8_begin();
    auto look = [&](uint32_t at) {
        mask = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < c.n_pages && c.refs[at + i] != 0u) mask |= 1u << i;
    };
    for (uint32_t base = 0; base < c.n_pages; base += 4 * kPlanThreads) {
        uint32_t total;
        look(base + 4 * threadIdx.x);
        block_scan(__popc(mask), sums, turn, &total);
        live += total;
    }
    // as many pages in use at or past `live` as free ones below it: the i-th goes to the i-th. A round has at most 4096 of either: one
    // scan adds up both, 16 bits each
    uint32_t holes = 0, movers = 0;
    for (uint32_t base = 0; base < c.n_pages; base += 4 * kPlanThreads) {
        const uint32_t at = base + 4 * threadIdx.x;
        if (c.n_pages > 4 * kPlanThreads) look(at);   // otherwise the one round above still stands
        uint32_t hole = 0, mover = 0, total;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < c.n_pages) {
                if (at + i < live && !(mask >> i & 1u)) hole |= 1u << i;
                if (at + i >= live && (mask >> i & 1u)) mover |= 1u << i;
                plan.slots[at + i] = at + i;
            }
        const uint32_t both = block_scan(__popc(hole) | __popc(mover) << 16, sums, turn, &total);
        uint32_t h = holes + (both & 0xffffu), m = movers + (both >> 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (hole >> i & 1u) plan.moves[h++].y = at + i;
            if (mover >> i & 1u) plan.moves[m++].x = at + i;
        }
        holes += total & 0xffffu;
        movers += total >> 16;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < movers; i += kPlanThreads) {
        const uint2 mv = plan.moves[i];
        plan.slots[mv.x] = mv.y;
        c.refs[mv.y] = c.refs[mv.x];
        c.refs[mv.x] = 0u;
    }
    if (threadIdx.x == 0) {
        plan.head[0] = movers;
        if (live_out) *live_out = live;
    }
}

// a = *quotient * b + remainder. Divided in 32 bits where it fits, which the units of a call nearly always do.
__device__ __forceinline__ uint32_t split(uint64_t a, uint32_t b, uint64_t* quotient) {
    if (a >> 32) {
        *quotient = a / b;
        return static_cast<uint32_t>(a % b);
    }
    const uint32_t q = static_cast<uint32_t>(a) / b;
    *quotient = q;
    return static_cast<uint32_t>(a) - q * b;
}

// Copies the listed pages in every layer; with `rename` also rewrites the table. A warp takes one (move, layer, K or V, head) at a time:
// page_size * hd codes and a scale. No page is both read and written (the lists are made so).
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(dc_kv8_cache c, Plan plan, bool rename, int* status) {
    const uint32_t lane = threadIdx.x & 31;
    kv8_begin();
    const uint64_t warps = static_cast<uint64_t>(gridDim.x) * (kCopyThreads / 32);
    const uint64_t units = static_cast<uint64_t>(plan.head[0]) * c.layers * 2 * c.nkv;
    const uint32_t row_bits = c.hd == 256 ? 4 : 3, in_row = (1u << row_bits) - 1, vectors = c.page_size << row_bits;   // a row of codes is 8 or 16 vectors
    const uint64_t first = static_cast<uint64_t>(blockIdx.x) * (kCopyThreads / 32) + (threadIdx.x >> 5);
    for (uint64_t u = first; u < units; u += warps) {
        uint64_t rest, move;
        const uint32_t head = split(u, c.nkv, &rest);
        const bool is_v = rest & 1u;
        const uint32_t layer = split(rest >> 1, c.layers, &move);
        const uint2 mv = plan.moves[move];
        uint8_t* base = static_cast<uint8_t*>(is_v ? c.v : c.k) + layer * c.layer_stride + head * c.head_stride;
        const uint8_t* from = base + mv.x * c.page_stride;
        uint8_t* to = base + mv.y * c.page_stride;
        for (uint32_t e = lane; e < vectors; e += 32 * 8) {   // eight requests in flight a lane
            uint4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = e + 32 * i;
                if (w < vectors) x[i] = *reinterpret_cast<const uint4*>(from + (w >> row_bits) * c.token_stride + 16 * (w & in_row));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = e + 32 * i;
                if (w < vectors) *reinterpret_cast<uint4*>(to + (w >> row_bits) * c.token_stride + 16 * (w & in_row)) = x[i];
            }
        }
        if (lane == 0) {
            float* scales = (is_v ? c.v_scale : c.k_scale) + static_cast<size_t>(layer) * c.n_pages * c.nkv + head;
            scales[static_cast<size_t>(mv.y) * c.nkv] = scales[static_cast<size_t>(mv.x) * c.nkv];
        }
    }
    if (!rename) return;
    for (uint64_t j = first; j < c.n_seqs; j += warps) {
        const uint32_t len = c.lens[j];
        if (!length_fits(c, len)) {
            if (lane == 0) kv8_flag(status, DC_STATUS_KV8_LENGTH);
            continue;
        }
        const uint32_t pages = kv8_pages(len, c.page_size);
        for (uint32_t col = lane; col < pages; col += 32) {
            uint32_t* at = c.table + j * c.max_pages + col;
            if (*at < c.n_pages) *at = plan.slots[*at];
            else kv8_flag(status, DC_STATUS_KV8_PAGE);
        }
    }
}

// The copying kernel's grid: up to `moves` pages will be listed, eight warps a CTA, at most eight CTAs an SM.
uint32_t copy_grid(const dc_ctx* ctx, const dc_kv8_cache* c, uint64_t moves) {
    const uint64_t units = moves * c->layers * 2 * c->nkv, ctas = (units + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
    const uint64_t most = static_cast<uint64_t>(ctx->sm_count) * 8;
    return static_cast<uint32_t>(ctas < 1 ? 1 : ctas < most ? ctas : most);
}

int pages_begin(dc_ctx* ctx, void* stream, const char* who, const dc_kv8_cache* cache, Plan* plan) {
    void* ws = nullptr;
    const int rc = dc_stream_workspace(ctx, static_cast<cudaStream_t>(stream), plan_bytes(cache->n_pages), who, &ws);
    if (rc == DC_OK) *plan = plan_at(ws, cache->n_pages);
    return rc;
}

}  // namespace

namespace {
int fail_text(char* err, size_t err_len, int code, const char* text) {
    if (err && err_len) snprintf(err, err_len, "%s", text);
    return code;
}
}  // namespace

extern "C" int dc_kv8_check(const dc_kv8_cache* c, char* err, size_t err_len) {
    if (err && err_len) err[0] = 0;
    if (!c) return fail_text(err, err_len, DC_INVALID_ARG, "null cache");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->table || !c->lens || !c->refs) return fail_text(err, err_len, DC_INVALID_ARG, "the cache has a null array");
    if (reinterpret_cast<uintptr_t>(c->k) % 16 || reinterpret_cast<uintptr_t>(c->v) % 16) return fail_text(err, err_len, DC_INVALID_ARG, "k and v must be 16-byte aligned");
    if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale) | reinterpret_cast<uintptr_t>(c->table) |
         reinterpret_cast<uintptr_t>(c->lens) | reinterpret_cast<uintptr_t>(c->refs)) % 4)
        return fail_text(err, err_len, DC_INVALID_ARG, "scales, table, lens and refs must be 4-byte aligned");
    if (c->hd != 128 && c->hd != 256) return fail_text(err, err_len, DC_UNSUPPORTED, "hd must be 128 or 256");
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return fail_text(err, err_len, DC_UNSUPPORTED, "page_size must be 16, 32, 64 or 128");
    if (!c->layers || !c->n_pages || !c->nkv || !c->n_seqs || !c->max_pages) return fail_text(err, err_len, DC_INVALID_ARG, "layers, n_pages, nkv, n_seqs and max_pages must be at least 1");
    if (c->n_seqs > 65535 || c->nkv > 1024 || c->layers > 65535) return fail_text(err, err_len, DC_UNSUPPORTED, "at most 65535 sequences, 65535 layers and 1024 kv heads");
    if (c->n_pages > 0x200000u) return fail_text(err, err_len, DC_UNSUPPORTED, "at most 2^21 pages");
    if (static_cast<uint64_t>(c->max_pages) * c->page_size >= 0x80000000ull) return fail_text(err, err_len, DC_UNSUPPORTED, "max_pages * page_size must be below 2^31");
    if (c->token_stride >= (1ull << 28)) return fail_text(err, err_len, DC_UNSUPPORTED, "token_stride must be below 2^28");
    if (c->reserved) return fail_text(err, err_len, DC_INVALID_ARG, "reserved must be 0");
    // codes must not share bytes: going up by stride, each step clears all that lies within the smaller ones
    uint64_t stride[4] = {c->token_stride, c->head_stride, c->page_stride, c->layer_stride}, count[4] = {c->page_size, c->nkv, c->n_pages, c->layers};
    uint64_t extent = c->hd;
    bool done[4] = {false, false, false, false};
    for (int i = 0; i < 4; ++i) {
        int least = -1;
        for (int k = 0; k < 4; ++k)
            if (!done[k] && (least < 0 || stride[k] < stride[least])) least = k;
        done[least] = true;
        if (count[least] == 1) continue;
        if (stride[least] % 16) return fail_text(err, err_len, DC_INVALID_ARG, "strides must be multiples of 16");
        if (stride[least] < extent) return fail_text(err, err_len, DC_INVALID_ARG, "strides make codes overlap");
        if (stride[least] > (1ull << 48) / count[least]) return fail_text(err, err_len, DC_INVALID_ARG, "strides pass 2^48 bytes");
        extent += stride[least] * (count[least] - 1);
    }
    return DC_OK;
}

int dc_kv8_require(dc_ctx* ctx, const char* who, const dc_kv8_cache* cache) {
    char text[160];
    const int rc = dc_kv8_check(cache, text, sizeof text);
    return rc == DC_OK ? DC_OK : dc_fail(ctx, rc, "%s: %s", who, text);
}

extern "C" size_t dc_kv8_pages_scratch_bytes(const dc_kv8_cache* cache) { return cache ? plan_bytes(cache->n_pages) : 0; }

extern "C" int dc_kv8_extend(dc_ctx* ctx, void* stream, const dc_kv8_cache* cache, const uint32_t* add) {
    if (!ctx) return DC_INVALID_ARG;
    int rc = dc_kv8_require(ctx, "kv8_extend", cache);
    if (rc != DC_OK) return rc;
    DC_REQUIRE(ctx, add, "kv8_extend: null operand");
    const dc_device_scope scope(ctx);
    Plan plan;
    if ((rc = pages_begin(ctx, stream, "kv8_extend", cache, &plan)) != DC_OK) return rc;
    return dc_kv8_launch(ctx, "kv8_extend", extend_kernel, true, dim3(1), kPlanThreads, 0, static_cast<cudaStream_t>(stream), *cache, add, plan, ctx->status_dev);
}

extern "C" int dc_kv8_fork(dc_ctx* ctx, void* stream, const dc_kv8_cache* cache, const uint32_t* src, const uint32_t* dst, uint32_t n, uint32_t deep) {
    if (!ctx) return DC_INVALID_ARG;
    int rc = dc_kv8_require(ctx, "kv8_fork", cache);
    if (rc != DC_OK) return rc;
    DC_REQUIRE(ctx, deep <= 1, "kv8_fork: deep = %u is neither 0 nor 1", deep);
    if (n == 0) return DC_OK;
    DC_REQUIRE(ctx, src && dst, "kv8_fork: null operand");
    DC_REQUIRE(ctx, n <= cache->n_seqs, "kv8_fork: %u forks of %u sequences", n, cache->n_seqs);
    const dc_device_scope scope(ctx);
    Plan plan;
    if ((rc = pages_begin(ctx, stream, "kv8_fork", cache, &plan)) != DC_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if ((rc = dc_kv8_launch(ctx, "kv8_fork", fork_kernel, true, dim3(1), kPlanThreads, (cache->n_seqs + 31) / 32 * 4, s, *cache, src, dst, n, deep != 0, plan, ctx->status_dev)) != DC_OK)
        return rc;
    const uint64_t most = deep ? static_cast<uint64_t>(n) * cache->max_pages : n;
    return dc_kv8_launch(ctx, "kv8_fork (copies)", copy_kernel, true, dim3(copy_grid(ctx, cache, most < cache->n_pages ? most : cache->n_pages)), kCopyThreads, 0, s, *cache, plan,
                         false, ctx->status_dev);
}

extern "C" int dc_kv8_free(dc_ctx* ctx, void* stream, const dc_kv8_cache* cache, const uint32_t* seqs, uint32_t n) {
    if (!ctx) return DC_INVALID_ARG;
    int rc = dc_kv8_require(ctx, "kv8_free", cache);
    if (rc != DC_OK) return rc;
    if (n == 0) return DC_OK;
    DC_REQUIRE(ctx, seqs, "kv8_free: null operand");
    const dc_device_scope scope(ctx);
    return dc_kv8_launch(ctx, "kv8_free", free_kernel, true, dim3(n), 128, 0, static_cast<cudaStream_t>(stream), *cache, seqs, ctx->status_dev);
}

extern "C" int dc_kv8_compact(dc_ctx* ctx, void* stream, const dc_kv8_cache* cache, uint32_t* live) {
    if (!ctx) return DC_INVALID_ARG;
    int rc = dc_kv8_require(ctx, "kv8_compact", cache);
    if (rc != DC_OK) return rc;
    const dc_device_scope scope(ctx);
    Plan plan;
    if ((rc = pages_begin(ctx, stream, "kv8_compact", cache, &plan)) != DC_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if ((rc = dc_kv8_launch(ctx, "kv8_compact", compact_kernel, true, dim3(1), kPlanThreads, 0, s, *cache, plan, live)) != DC_OK) return rc;
    // at most half of the pages move
    return dc_kv8_launch(ctx, "kv8_compact (copies)", copy_kernel, true, dim3(copy_grid(ctx, cache, cache->n_pages / 2 + 1)), kCopyThreads, 0, s, *cache, plan, true, ctx->status_dev);
}
