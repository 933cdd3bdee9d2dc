// The work list of one step's paged attention, made once and read by the
// attention of every layer.
//
// One workgroup.  A request of n new tokens has n * group rows per KV head;
// they are cut into units of up to 32, 64 or 128 rows that walk the request's
// key tiles together.  Larger units read each key tile for more rows, smaller
// ones spread better: the size is the largest that gives every lane (a
// workgroup of the attention kernel) two units, or, for fewer rows than that,
// the largest whose tiles, split over all lanes, still make a walk of
// kWalkTiles each.  A unit that costs more than `cap` is split over its key
// tiles into items with partial results.  `cap` is the candidate with the
// least estimated time: the rounds of items per lane times the longest, against
// the even share plus the longest.  The items are ordered by cost, longest
// first, and lane l takes items l, 2N-1-l, 2N+l, ... of N lanes.
//
// Costs are in quarters of the time in which one lane runs a 64-key tile of 32
// rows out of the cache: the products of 32 rows take 4, and the tile's bytes
// from HBM kHbmCost, shared by the units of the request that read them.
#include "common.hpp"
#include "paged.hpp"

namespace tiattn {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr uint32_t kHbmCost = 16;
constexpr uint32_t kItemCost = 16;   // starting and merging an item
constexpr uint32_t kWalkTiles = 8;
constexpr int kCaps = 32;
// Candidates for `cap` over the even share per lane, the last unbounded.  At
// least half of it, which bounds the partial results (paged_partial_blocks).
__device__ const float kCapOver[kCaps] = {1.0f,  1.02f, 1.04f, 1.06f, 1.08f, 1.1f,  1.13f, 1.16f,
                                          1.2f,  1.25f, 1.3f,  1.35f, 1.4f,  1.5f,  1.6f,  1.75f,
                                          1.9f,  2.0f,  2.2f,  2.5f,  2.75f, 3.0f,  3.5f,  4.0f,
                                          5.0f,  6.0f,  8.0f,  10.0f, 12.0f, 16.0f, 32.0f, 3.0e38f};

__device__ __forceinline__ uint64_t wave_sum64(uint64_t x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m);
    return x;
}
__device__ __forceinline__ uint32_t wave_max32(uint32_t x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x = max(x, (uint32_t)__shfl_xor(x, m));
    return x;
}

// Exclusive sum over the workgroup's threads in thread order, total in *sum.
__device__ __forceinline__ uint32_t block_scan(uint32_t x, uint32_t* sum) {
    __shared__ uint32_t s_tot[kPlanWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t inc = x;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const uint32_t u = __shfl_up(inc, m);
        if (lane >= m) inc += u;
    }
    if (lane == 63) s_tot[wave] = inc;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        before += w < wave ? s_tot[w] : 0;
        all += s_tot[w];
    }
    __syncthreads();
    *sum = all;
    return before + inc - x;
}

__device__ __forceinline__ uint64_t block_sum64(uint64_t x) {
    __shared__ uint64_t s_tot[kPlanWaves];
    x = wave_sum64(x);
    if ((threadIdx.x & 63) == 0) s_tot[threadIdx.x >> 6] = x;
    __syncthreads();
    uint64_t r = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) r += s_tot[w];
    __syncthreads();
    return r;
}

__device__ __forceinline__ uint32_t unit_rows_for(uint32_t rows) { return rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

struct Request {
    uint32_t token0, n, len;
};
// Lengths as the kernels may use them whatever the arrays hold: tokens inside
// q, keys inside the block table.
__device__ __forceinline__ Request request(const PagedPlanArgs& a, uint32_t b) {
    Request r;
    const uint32_t s = min(a.query_start[b], a.head.num_tokens), e = min(a.query_start[b + 1], a.head.num_tokens);
    const uint64_t room = (uint64_t)a.head.max_blocks * a.head.page_size;
    r.token0 = s;
    r.n = e > s ? e - s : 0;
    r.len = (uint32_t)min((uint64_t)a.seq_lens[b], room);
    return r;
}

// The key tiles that rows [row0, row0 + rows) see (tile_end = their number).
__device__ __forceinline__ PagedItem unit_of(const PagedPlanArgs& a, uint32_t b, const Request& r, uint32_t group,
                                             uint32_t row0, uint32_t rows) {
    PagedItem u;
    u.req = b;
    u.token0 = r.token0;
    u.row0 = row0;
    u.rows = rows;
    u.pos0 = (int32_t)r.len - (int32_t)r.n;
    const int32_t first = u.pos0 + (int32_t)(row0 / group), last = u.pos0 + (int32_t)((row0 + rows - 1) / group);
    u.key_end = last < 0 ? 0 : (uint32_t)last + 1;
    uint32_t low = 0;
    if (a.head.window && first >= 0 && (uint32_t)first + 1 > a.head.window) low = (uint32_t)first + 1 - a.head.window;
    u.low_tile = low / kPagedTile;
    const uint32_t sink_tiles = (uint32_t)(((uint64_t)a.head.sinks + kPagedTile - 1) / kPagedTile);
    u.sink_tiles = a.head.window ? min(sink_tiles, u.low_tile) : 0;
    u.tile_begin = 0;
    u.tile_end = u.key_end ? (u.key_end - 1) / kPagedTile + 1 - u.low_tile + u.sink_tiles : 0;
    u.partial = kPagedWhole;
    u.pad = 0;
    return u;
}

__device__ __forceinline__ uint32_t tile_cost(uint32_t rows, uint32_t units) {
    const uint32_t compute = rows <= 32 ? 4 : rows <= 64 ? 8 : 16;
    return max(compute, kHbmCost / units);
}

// Pieces of a unit of `tiles` tiles and cost `cost` under `cap`.  Units of up
// to 32 rows are split in pairs of tiles, one 32-key half per wave.
__device__ __forceinline__ uint32_t pieces_of(uint32_t cost, uint32_t tiles, uint32_t rows, float inv_cap) {
    const uint32_t most = rows <= 32 ? (tiles + 1) / 2 : tiles;
    const float want = ceilf((float)cost * inv_cap - 1e-3f);
    return want <= 1.0f ? 1 : min((uint32_t)fminf(want, 65536.0f), max(most, 1u));
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedPlanArgs a) {
    constexpr uint32_t kBuckets = 1024;
    __shared__ uint32_t s_first[kPagedMaxBatch + 1];  // first unit of each request
    __shared__ uint32_t s_bucket[kBuckets];
    __shared__ float s_est[kCaps];
    __shared__ uint32_t s_pick;
    const uint32_t tid = threadIdx.x, batch = a.head.batch, hkv = a.head.hkv, group = a.head.hq / hkv;
    const uint32_t lanes = paged_lanes(hkv), max_units = paged_max_units(batch, a.head.num_tokens, group);
    const PagedPlanLayout lay = paged_plan_layout(batch, a.head.num_tokens, a.head.hq, hkv);
    char* const base = static_cast<char*>(a.plan);
    PagedItem* const items = reinterpret_cast<PagedItem*>(base + lay.items);
    PagedItem* const units = reinterpret_cast<PagedItem*>(base + lay.units);
    PagedSplitBlock* const split = reinterpret_cast<PagedSplitBlock*>(base + lay.split_blocks);
    uint32_t* const costs = reinterpret_cast<uint32_t*>(base + lay.costs);
    uint32_t* const offsets = costs + max_units + 1;

    // Rows per unit.
    uint64_t n_units[3] = {0, 0, 0}, n_tiles[3] = {0, 0, 0};
    for (uint32_t b = tid; b < batch; b += kPlanThreads) {
        const Request r = request(a, b);
        const uint32_t rows = r.n * group;
        if (!rows) continue;
        // The tiles that the request's middle rows see.
        const PagedItem mid = unit_of(a, b, r, group, rows / 2, 1);
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const uint32_t R = min(32u << i, unit_rows_for(rows));
            n_units[i] += (rows + R - 1) / R;
            n_tiles[i] += (uint64_t)((rows + R - 1) / R) * mid.tile_end;
        }
    }
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        n_units[i] = block_sum64(n_units[i]);
        n_tiles[i] = block_sum64(n_tiles[i]);
    }
    uint32_t unit_rows = 32;
    if (n_units[2] >= 2 * lanes) unit_rows = 128;
    else if (n_units[1] >= 2 * lanes) unit_rows = 64;
    else if (n_units[0] >= 2 * lanes) unit_rows = 32;
    else if (n_tiles[2] >= (uint64_t)kWalkTiles * lanes) unit_rows = 128;
    else if (n_tiles[1] >= (uint64_t)kWalkTiles * lanes) unit_rows = 64;

    // The units.
    uint32_t U = 0;
    for (uint32_t b0 = 0; b0 < batch; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        uint32_t n = 0, sum;
        if (b < batch) {
            const uint32_t rows = request(a, b).n * group, R = min(unit_rows, unit_rows_for(rows));
            n = (rows + R - 1) / R;
        }
        // The bound holds for any ascending query_start; it also keeps units
        // of an array that is none inside the plan.
        const uint32_t at = block_scan(n, &sum);
        if (b < batch) s_first[b] = min(U + at, max_units);
        U = min(U + sum, max_units);
    }
    if (tid == 0) s_first[batch] = U;
    __syncthreads();
    uint64_t my_cost = 0;
    uint32_t my_max = 0;
    for (uint32_t i = tid; i < U; i += kPlanThreads) {
        uint32_t lo = 0, hi = batch;  // s_first[lo] <= i < s_first[hi]
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (s_first[mid] <= i)
                lo = mid;
            else
                hi = mid;
        }
        const Request r = request(a, lo);
        const uint32_t rows = r.n * group, R = min(unit_rows, unit_rows_for(rows)), row0 = (i - s_first[lo]) * R;
        const PagedItem u = unit_of(a, lo, r, group, row0, min(R, rows - row0));
        const uint32_t cost = u.tile_end * tile_cost(u.rows, s_first[lo + 1] - s_first[lo]) + kItemCost;
        units[i] = u;
        costs[i] = cost;
        my_cost += cost;
        my_max = max(my_max, cost);
    }
    const uint64_t work = block_sum64(my_cost);  // (also orders units and costs)
    const float share = (float)work / lanes;

    // Each wave estimates two candidates for the cap.
    const int lane = tid & 63, wave = tid >> 6;
    for (int k = wave; k < kCaps; k += kPlanWaves) {
        const float inv_cap = kCapOver[k] > 1.0e30f ? 0.0f : 1.0f / (kCapOver[k] * share);
        uint64_t n = 0;
        uint32_t longest = 0;
        for (uint32_t i = lane; i < U; i += 64) {
            const uint32_t tiles = units[i].tile_end, p = pieces_of(costs[i], tiles, units[i].rows, inv_cap);
            n += p;
            longest = max(longest, (costs[i] - kItemCost) / p + (p > 1 ? 1 : 0) + kItemCost);
        }
        n = wave_sum64(n);
        longest = wave_max32(longest);
        const float rounds = ceilf((float)n / lanes);
        const float even = share + (float)(n - U) * kItemCost / lanes + (float)longest;
        if (lane == 0) s_est[k] = fminf(rounds * longest, even);
    }
    __syncthreads();
    if (tid == 0) {
        uint32_t best = kCaps - 1;
        for (int k = kCaps - 2; k >= 0; --k)
            if (s_est[k] < s_est[best]) best = k;
        s_pick = best;
    }
    for (uint32_t i = tid; i < kBuckets; i += kPlanThreads) s_bucket[i] = 0;
    __syncthreads();
    const uint32_t pick = s_pick;
    const float inv_cap = kCapOver[pick] > 1.0e30f ? 0.0f : 1.0f / (kCapOver[pick] * share);

    // Items and partial blocks of each unit: offsets[i] = first item, and the
    // unit's `partial` = its first partial block.
    uint32_t N = 0, blocks = 0, split_blocks = 0;
    uint32_t longest = 0;
    for (uint32_t i0 = 0; i0 < U; i0 += kPlanThreads) {
        const uint32_t i = i0 + tid;
        uint32_t p = 0, nb = 0, sum;
        PagedItem u{};
        if (i < U) {
            u = units[i];
            p = pieces_of(costs[i], u.tile_end, u.rows, inv_cap);
            nb = (u.rows + kPagedBlockRows - 1) / kPagedBlockRows;
            longest = max(longest, costs[i] / p);
        }
        const uint32_t at = block_scan(p, &sum);
        if (i < U) offsets[i] = N + at;
        N += sum;
        const uint32_t pb = block_scan(p > 1 ? p * nb : 0, &sum), first = blocks + pb;
        blocks += sum;
        const uint32_t sb = block_scan(p > 1 ? nb : 0, &sum);
        if (p > 1) {
            units[i].partial = first;
            for (uint32_t k = 0; k < nb; ++k) {
                PagedSplitBlock s{};
                s.token0 = u.token0;
                s.row0 = u.row0 + k * kPagedBlockRows;
                s.rows = min(kPagedBlockRows, u.rows - k * kPagedBlockRows);
                s.first = first + k;
                s.stride = nb;
                s.pieces = p;
                split[split_blocks + sb + k] = s;
            }
        }
        split_blocks += sum;
    }
    __shared__ uint32_t s_max[kPlanWaves];
    longest = wave_max32(longest);
    if (lane == 0) s_max[wave] = longest;
    if (tid == 0) offsets[U] = N;
    __syncthreads();
    longest = 1;
    for (int w = 0; w < kPlanWaves; ++w) longest = max(longest, s_max[w]);

    // The items, longest first (by cost buckets; order within a bucket decides
    // only which lane runs an item, never a result).
    const float to_bucket = (float)(kBuckets - 1) / (float)longest;
    for (int pass = 0; pass < 2; ++pass) {
        for (uint32_t i = tid; i < N; i += kPlanThreads) {
            uint32_t lo = 0, hi = U;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                if (offsets[mid] <= i)
                    lo = mid;
                else
                    hi = mid;
            }
            const uint32_t p = offsets[lo + 1] - offsets[lo], k = i - offsets[lo];
            const uint32_t bucket = kBuckets - 1 - min(kBuckets - 1, (uint32_t)((float)(costs[lo] / p) * to_bucket));
            if (pass == 0) {
                atomicAdd(&s_bucket[bucket], 1u);
            } else {
                PagedItem u = units[lo];
                if (p > 1) {
                    const uint32_t nb = (u.rows + kPagedBlockRows - 1) / kPagedBlockRows;
                    const uint32_t quantum = u.rows <= 32 ? 2 : 1, q = (u.tile_end + quantum - 1) / quantum;
                    const uint32_t tiles = u.tile_end;
                    u.tile_begin = quantum * (uint32_t)((uint64_t)q * k / p);
                    u.tile_end = min(tiles, quantum * (uint32_t)((uint64_t)q * (k + 1) / p));
                    u.partial += k * nb;
                }
                items[atomicAdd(&s_bucket[bucket], 1u)] = u;
            }
        }
        __syncthreads();
        if (pass == 0) {
            uint32_t sum;
            const uint32_t c = s_bucket[tid];
            const uint32_t at = block_scan(c, &sum);
            s_bucket[tid] = at;
            __syncthreads();
        }
    }
    static_assert(kBuckets == kPlanThreads, "one bucket per thread in the scan");
    if (tid == 0) {
        PagedPlanHeader h = a.head;
        h.magic = kPagedMagic;
        h.units = U;
        h.items = N;
        h.split_blocks = split_blocks;
        *reinterpret_cast<PagedPlanHeader*>(base) = h;
    }
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace tiattn
