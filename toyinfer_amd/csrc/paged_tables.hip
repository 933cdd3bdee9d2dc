// A serving step's bookkeeping and its first pass over a layer's rows.
//
// Tables.  Request b has c cached tokens and n new ones.  Its block table
// grows from ceil(c / ps) to ceil((c + n) / ps) pages, taken from the top of a
// stack of free pages in request order: an exclusive sum of the needs says
// which.  New token i gets position c + i and the slot (page, row in page) of
// that position.  The step moves a few bytes per token; what it costs is one
// launch and the chain lengths -> sums -> tables -> slots, so every workgroup
// repeats the sums over the requests (a few words each) instead of waiting for
// another one's, and the tokens are spread over the grid.  A new token's page
// is found from the sums, never through the table entry that this launch
// writes.  8 requests take 3.2 us, 200 with 1300 tokens 4.3, of which a launch
// with nothing to do is about 2.
//
// Prologue.  Per row of D: y = x / sqrt(mean(x^2) + eps) * w, rotated by the
// position's (cos, sin), rounded once to bf16; Q goes to its buffer, K and V to
// their cache slots.  Bound by memory: each row is read and written once.
#include <math.h>

#include "common.hpp"
#include "paged.hpp"
#include "paged_rows.hpp"

namespace tiattn {
namespace {

constexpr int kTabThreads = 256;
constexpr uint32_t kTabTokens = 1024;  // token rows per workgroup
constexpr uint32_t kTabMaxWgs = 256;

// Exclusive sums over the workgroup's threads, in thread order; the totals in
// *sum_a, *sum_b.
__device__ __forceinline__ void block_scan2(uint64_t& a, uint64_t& b, uint64_t* sum_a, uint64_t* sum_b) {
    constexpr int NW = kTabThreads / 64;
    __shared__ uint64_t s_tot[NW][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t ia = wave_scan(a, Sum{}), ib = wave_scan(b, Sum{});
    if (lane == 63) {
        s_tot[wave][0] = ia;
        s_tot[wave][1] = ib;
    }
    __syncthreads();
    uint64_t ta = 0, tb = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        if (w == wave) {
            a = ta + ia - a;
            b = tb + ib - b;
        }
        ta += s_tot[w][0];
        tb += s_tot[w][1];
    }
    *sum_a = ta;
    *sum_b = tb;
    __syncthreads();
}

__device__ __forceinline__ uint32_t clamp32(uint64_t x) { return x > 0xffffffffull ? 0xffffffffu : (uint32_t)x; }

__global__ __launch_bounds__(kTabThreads) void paged_tables_kernel(PagedTablesArgs a) {
    __shared__ uint32_t s_start[kPagedMaxBatch + 1];  // first token row
    __shared__ uint32_t s_first[kPagedMaxBatch];      // its first page counted down the stack, kNoSlot: refused
    const uint32_t tid = threadIdx.x, page_size = 1u << a.page_shift;
    const uint32_t num_free = min(*a.num_free, a.free_capacity);

    uint64_t tokens = 0, pages = 0;   // of the requests before this round's
    uint64_t taken = 0, refused = 0;  // of this thread's requests
    for (uint32_t b0 = 0; b0 < a.batch; b0 += kTabThreads) {
        const uint32_t b = b0 + tid;
        const bool has = b < a.batch;
        const uint64_t c = has ? a.context_lens[b] : 0, n = has ? a.new_lens[b] : 0;
        const uint64_t old = (c + page_size - 1) >> a.page_shift;
        const uint64_t end = (c + n + page_size - 1) >> a.page_shift;
        const uint64_t need = end <= a.max_blocks ? end - old : 0;
        uint64_t st = n, first = need, sum_n, sum_p;
        block_scan2(st, first, &sum_n, &sum_p);
        st += tokens;
        first += pages;
        tokens += sum_n;
        pages += sum_p;
        if (has) {
            // (A request without new tokens has no rows that could pass num_tokens.)
            const bool ok = end <= a.max_blocks && (n == 0 || st + n <= a.num_tokens) &&
                            (need == 0 || first + need <= num_free);
            s_start[b] = clamp32(st);
            s_first[b] = ok ? (uint32_t)(need ? first : 0) : kNoSlot;
            if (ok) taken = max(taken, need ? first + need : 0);
            refused += !ok;
            if (blockIdx.x == 0) {
                a.query_start[b] = clamp32(st);
                a.seq_lens[b] = clamp32(ok ? c + n : c);
            }
        }
    }
    if (tid == 0) s_start[a.batch] = clamp32(tokens);
    __syncthreads();
    if (blockIdx.x == 0) {
        // Accepted requests that need pages are a prefix of those that do, so
        // the pages taken are the largest end among them.
        __shared__ uint32_t s_taken[kTabThreads / 64];
        const uint32_t most = wave_scan((uint32_t)taken, Max{});
        if ((tid & 63) == 63) s_taken[tid >> 6] = most;
        uint64_t unused = 0, sum_r, sum_u;
        block_scan2(refused, unused, &sum_r, &sum_u);
        if (tid == 0) {
            a.query_start[a.batch] = clamp32(tokens);
            uint32_t all = 0;
#pragma unroll
            for (int w = 0; w < kTabThreads / 64; ++w) all = max(all, s_taken[w]);
            a.status[0] = num_free - all;
            a.status[1] = (uint32_t)sum_r;
        }
    }

    // The new entries of the block tables, a wave per request.
    const uint32_t lane = tid & 63, waves = gridDim.x * (kTabThreads / 64);
    for (uint32_t b = blockIdx.x * (kTabThreads / 64) + (tid >> 6); b < a.batch; b += waves) {
        const uint32_t first = s_first[b];
        if (first == kNoSlot) continue;
        const uint32_t c = a.context_lens[b], n = s_start[b + 1] - s_start[b];
        const uint32_t old = (uint32_t)(((uint64_t)c + page_size - 1) >> a.page_shift);
        const uint32_t end = (uint32_t)(((uint64_t)c + n + page_size - 1) >> a.page_shift);
        for (uint32_t j = old + lane; j < end; j += 64)
            a.block_tables[(uint64_t)b * a.max_blocks + j] = a.free_pages[num_free - 1 - first - (j - old)];
    }

    // Positions and slots.
    const uint32_t total = s_start[a.batch];
    for (uint32_t t = blockIdx.x * kTabThreads + tid; t < a.num_tokens; t += gridDim.x * kTabThreads) {
        uint32_t pos = 0, slot = kNoSlot;
        if (t < total) {
            uint32_t lo = 0, hi = a.batch;  // s_start[lo] <= t < s_start[hi]
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (s_start[mid] <= t)
                    lo = mid;
                else
                    hi = mid;
            }
            const uint32_t c = a.context_lens[lo], first = s_first[lo];
            pos = c + (t - s_start[lo]);
            if (first != kNoSlot) {
                const uint32_t old = (uint32_t)(((uint64_t)c + page_size - 1) >> a.page_shift);
                const uint32_t j = pos >> a.page_shift;
                const uint32_t page = j < old ? a.block_tables[(uint64_t)lo * a.max_blocks + j]
                                              : a.free_pages[num_free - 1 - first - (j - old)];
                const uint64_t s = ((uint64_t)page << a.page_shift) + (pos & (page_size - 1));
                slot = s < kNoSlot ? (uint32_t)s : kNoSlot;
            }
        }
        a.positions[t] = pos;
        a.slots[t] = slot;
    }
}

// D / 16 lanes per row, lane c the eight pairs (8c + k, 8c + k + D/2); a wave has
// G consecutive rows of a token.  Each input row is read once and each output row
// written once, and both bypass the caches' retention: 8192 tokens of 32 + 2 * 8 heads
// 40.2 -> 36.6 us (5.5 TB/s, the rate of a large copy).  Two and four rows per lane
// group, to read a position's angles and the weights once for them, gave up to 2 % on
// 8192 tokens and cost a small call 0.3 and 1.1 us of 2.5.
template <int D>
__global__ __launch_bounds__(256) void paged_prologue_kernel(PagedPrologueArgs a, uint32_t parts) {
    constexpr int LPR = D / 16, G = 64 / LPR, HALF = D / 2;
    const uint32_t unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t t = unit / parts, part = unit % parts;
    if (t >= a.num_tokens) return;
    const int lane = threadIdx.x & 63, c = lane % LPR;
    // Row j of the token: of q, then k, then v; past the last one: that.
    const uint32_t rows = a.hq + 2 * a.hkv, row = part * G + lane / LPR, j = min(row, rows - 1);
    const bool is_q = j < a.hq, is_k = !is_q && j < a.hq + a.hkv;
    const uint32_t heads = is_q ? a.hq : a.hkv, head = j - (is_q ? 0 : is_k ? a.hq : a.hq + a.hkv);
    const uint32_t pos = min(a.positions[t], a.num_positions - 1);
    const uint32_t slot = a.slots[t];
    const uint64_t at = ((uint64_t)t * heads + head) * D;
    const uint16_t* src = (is_q ? a.q : is_k ? a.k : a.v) + at;
    uint4 xr = ldg16_nt(src + 8 * c), xi = ldg16_nt(src + 8 * c + HALF);
    const uint4 qwr = ldg16(a.q_weight + 8 * c), qwi = ldg16(a.q_weight + 8 * c + HALF);
    const uint4 kwr = ldg16(a.k_weight + 8 * c), kwi = ldg16(a.k_weight + 8 * c + HALF);
    float4 cs[4];
    const float4* rope = reinterpret_cast<const float4*>(a.rope + (uint64_t)pos * D + 16 * c);
#pragma unroll
    for (int k = 0; k < 4; ++k) cs[k] = rope[k];
    const uint64_t cache_row = (uint64_t)(slot >> a.page_shift) * a.page_stride +
                               (uint64_t)(slot & ((1u << a.page_shift) - 1)) * a.hkv * D;
    if (is_q || is_k) {
        float re[8], im[8];
        norm_rope_f32<D>(xr, xi, is_q ? qwr : kwr, is_q ? qwi : kwi, cs, a.eps, re, im);
        xr = pack_bf16x8(re);
        xi = pack_bf16x8(im);
    }
    if (row < rows && (is_q || slot < a.num_slots)) {
        uint16_t* dst = (is_q ? a.q_out : is_k ? a.k_cache : a.v_cache) + (is_q ? at : cache_row + (uint64_t)head * D);
        stg16_nt(dst + 8 * c, xr);
        stg16_nt(dst + 8 * c + HALF, xi);
    }
}

template <int D>
hipError_t launch_prologue_t(const PagedPrologueArgs& a, hipStream_t st) {
    constexpr uint32_t G = 64 / (D / 16);
    const uint32_t parts = (a.hq + 2 * a.hkv + G - 1) / G;
    const uint64_t units = (uint64_t)a.num_tokens * parts;
    hipLaunchKernelGGL((paged_prologue_kernel<D>), dim3((uint32_t)((units + 3) / 4)), dim3(256), 0, st, a, parts);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_tables(const PagedTablesArgs& a, hipStream_t stream) {
    const uint32_t by_tokens = (a.num_tokens + kTabTokens - 1) / kTabTokens;
    const uint32_t by_requests = (a.batch + 3) / 4;
    const uint32_t wgs = min(kTabMaxWgs, max(by_tokens, by_requests));
    hipLaunchKernelGGL(paged_tables_kernel, dim3(wgs), dim3(kTabThreads), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_paged_prologue(const PagedPrologueArgs& a, uint32_t d, hipStream_t stream) {
    return d == 64 ? launch_prologue_t<64>(a, stream) : launch_prologue_t<128>(a, stream);
}

}  // namespace tiattn
