// The work list of one step's paged attention, made once and read by the
// attention of every layer.
//
// One workgroup.  A request of n new tokens has n * group rows per KV head;
// they are cut into units of up to 32, 64, 128 or 256 rows that walk the request's
// key tiles together.  Larger units read each key tile for more rows, smaller
// ones spread better over the lanes (a lane: a workgroup of the attention
// kernel).  Either
// * each unit is a list, longest first, and the lanes draw lists as they come
//   free, or
// * the units' tiles laid end to end are cut into ranges, one per lane of its even
//   share; or, with units of 64 or 128 rows, of 7/8 of it, and as many of 1/8 that
//   the lanes draw afterwards, for their speeds differ.  A unit with a cut inside
//   leaves partial results of each piece, merged by a second kernel.
// Streamed requests take even shares only: every range more is a piece more to
// start and merge (32 requests of 8192 keys 167 us, 179 with the two ranges and
// 180 with whole requests; mixed batches with units of 128 rows are 1 to 7 %
// faster with the two).
// The size and the way are those with the shortest estimate: rounds of whole
// units times their mean, or the longest of them, against the even share plus
// the pieces' overhead.  Forced ones took, in us, at 32 query and 8 KV heads of
// 128 (w whole, c cut, * the choice):
//                              64 w / c     128 w / c    256 w / c rows
//   512 tokens on 8192 keys    93 / 123     119 / 82*    204 / 83
//   a prompt of 512            16* / 23      20 / 23      26 / 28
//   a prompt of 2048           76 / 83       66* / 73     64 / 70
//   a prompt of 8192          757 / 800     587 / 662    533* / 580
//   30 decoded and 5 chunks   182 / 211     156 / 174    181 / 158*
// (32 rows: 201 for the first and 1494 for the fourth.)
//
// One workgroup, because each phase needs the sums of the one before: 9.4 us for
// 32 requests, 15.7 for 1000, once per step; half of it are waits for memory and
// between phases.
//
// Costs are in units of about 0.12 us of a lane.  A 64-key tile takes its
// products (up to 32 rows: the latency of its bytes), or, for requests of up to
// 32 rows in a step bound by the keys' bytes, its share of the bandwidth.
#include "common.hpp"
#include "paged.hpp"

namespace tiattn {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr uint32_t kStreamTile = 8;  // of up to 32 rows: the latency of its bytes, at either head_dim
constexpr uint32_t kStreamItem = 24, kSharedItem = 80;  // starting and finishing an item
constexpr uint32_t kPieceTiles = 2;  // cuts lie on multiples of it, one 32-key half per wave
constexpr uint32_t kLocalUnits = 2048;
constexpr uint32_t kSizes = 4;         // of units: 32, 64, 128 or 256 rows
constexpr uint32_t kTwoRanges = 500;   // a lane's share from which it is in two ranges

// Exclusive sums over the workgroup's threads in thread order, total in *sum.
template <typename T>
__device__ __forceinline__ T block_scan(T x, T* sum) {
    __shared__ T s_tot[kPlanWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T inc = wave_scan(x, Sum{});
    if (lane == 63) s_tot[wave] = inc;
    __syncthreads();
    T before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        before += w < wave ? s_tot[w] : 0;
        all += s_tot[w];
    }
    __syncthreads();
    *sum = all;
    return before + inc - x;
}

// Index of the last entry <= x of ascending a[0..n), a[0] <= x.
template <typename T>
__device__ __forceinline__ uint32_t last_at_most(const T* a, uint32_t n, T x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (a[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// Unit sizes are 32 << index.
__device__ __forceinline__ uint32_t size_for(uint32_t rows) { return (rows > 32) + (rows > 64) + (rows > 128); }

struct Request {
    uint32_t token0, n, len;
};

// The key tiles that rows [row0, row0 + rows) of request b see.
__device__ __forceinline__ PagedItem unit_of(const PagedPlanHeader& h, uint32_t b, const Request& r, uint32_t group,
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
    if (h.window && first >= 0 && (uint32_t)first + 1 > h.window) low = (uint32_t)first + 1 - h.window;
    u.low_tile = low / kPagedTile;
    const uint32_t sink_tiles = (uint32_t)(((uint64_t)h.sinks + kPagedTile - 1) / kPagedTile);
    u.sink_tiles = h.window ? min(sink_tiles, u.low_tile) : 0;
    u.tile_begin = 0;
    u.tile_end = u.key_end ? (u.key_end - 1) / kPagedTile + 1 - u.low_tile + u.sink_tiles : 0;
    u.partial = kPagedWhole;
    u.next = kPagedNone;
    return u;
}

// A tile's products, by the unit's rows (at head_dim 64 less than at 128, but not
// in a batch with streamed requests: with two thirds there, mixed ones took 7 to
// 15 % longer, and prompts of 512 to 8192 tokens the same within 1 %); its bytes' time
// where all lanes stream at once.
__device__ __forceinline__ uint32_t product_cost(uint32_t rows) {
    return rows <= 32 ? kStreamTile : rows <= 64 ? 6 : rows <= 128 ? 9 : 17;
}
__device__ __forceinline__ uint32_t bytes_cost(uint32_t d) { return d == 64 ? 6 : 11; }
// Of a request with up to 32 rows in a step that streams.
__device__ __forceinline__ uint32_t stream_cost(uint32_t d) { return max(kStreamTile, bytes_cost(d)); }
__device__ __forceinline__ uint32_t item_cost(uint32_t rows) { return rows <= 32 ? kStreamItem : kSharedItem; }

// The whole step, for U units of this total and longest cost: each as a list of
// its own, or cut into even shares.  `streamed`: the cost of the units of
// requests with up to 32 rows.
struct Estimate {
    uint64_t whole, cut;
    uint32_t levels;
};
__device__ __forceinline__ Estimate estimate(uint32_t U, uint64_t work, uint64_t longest, uint64_t streamed,
                                             uint32_t rows, uint32_t lanes) {
    const uint64_t share = work / lanes;
    Estimate e;
    e.levels = (rows == 64 || rows == 128) && share >= kTwoRanges ? kPagedLevels : 1;
    const uint64_t rounds = U ? (uint64_t)((U + lanes - 1) / lanes) * work / U : 0;
    e.whole = max(longest, rounds) + (rows == 32 ? longest / 4 : 0);
    // A cut costs a lane another item and its piece's results (half a unit per
    // row), by what it falls into.
    const float in_stream = rows == 32 || !work ? 1.0f : (float)streamed / (float)work;
    const float per_cut = in_stream * (item_cost(32) + 16) + (1.0f - in_stream) * (item_cost(rows) + rows / 2);
    e.cut = share + 8 + (uint64_t)(per_cut * e.levels);
    return e;
}

// Sizes of a lane's ranges, in parts of its share.
constexpr uint32_t kParts = 16, kFirstParts = 14;

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedPlanArgs a) {
    constexpr uint32_t kBuckets = kPlanThreads;
    __shared__ Request s_req[kPagedMaxBatch];
    __shared__ uint32_t s_first[kPagedMaxBatch + 1];   // first unit of each request
    __shared__ uint64_t s_cost[kLocalUnits + 1];       // cost of the units before each
    __shared__ uint32_t s_cut_unit[kPagedLevels * kPagedSlots + 1], s_cut_tile[kPagedLevels * kPagedSlots + 1];
    __shared__ uint32_t s_item[kPagedLevels * kPagedSlots + 1];  // first item of each range
    __shared__ PagedItem s_unit[kPlanThreads];  // the first units, as in the plan
    __shared__ uint32_t s_bucket[kBuckets];
    __shared__ uint64_t s_work[kPlanWaves][kSizes];
    __shared__ uint32_t s_units[kPlanWaves][kSizes], s_long[kPlanWaves][kSizes], s_most[kPlanWaves];
    __shared__ uint64_t s_time[kSizes], s_bytes[kPlanWaves], s_products[kPlanWaves], s_streamed[kPlanWaves + 1];
    __shared__ uint32_t s_streams[kPlanWaves + 1], s_stream_long[kPlanWaves];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t batch = a.head.batch, hkv = a.head.hkv, group = a.head.hq / hkv;
    const uint32_t lanes = paged_lanes(hkv), max_units = paged_max_units(batch, a.head.num_tokens, group);
    const PagedPlanLayout lay = paged_plan_layout(batch, a.head.num_tokens, a.head.hq, hkv);
    char* const base = static_cast<char*>(a.plan);
    PagedItem* const items = reinterpret_cast<PagedItem*>(base + lay.items);
    PagedItem* const units = reinterpret_cast<PagedItem*>(base + lay.units);
    PagedSplitBlock* const split = reinterpret_cast<PagedSplitBlock*>(base + lay.split_blocks);

    // Lengths as the kernels may use them whatever the arrays hold: tokens
    // inside q, keys inside the block table.  For each size its units, their
    // cost (by the request's middle unit) and the longest (by its last).  The
    // step streams if its keys' bytes take longer than its products: then each
    // lane gets its share of the bandwidth, and else as much as it asks for.
    uint64_t work_of[kSizes] = {}, bytes = 0, products = 0, streamed = 0;
    uint32_t units_of[kSizes] = {}, long_of[kSizes] = {}, most = 0, stream_long = 0, streams = 0;
    const uint32_t room = (uint32_t)min((uint64_t)a.head.max_blocks * a.head.page_size, (uint64_t)0x7fffffffu);
    for (uint32_t b = tid; b < batch; b += kPlanThreads) {
        const uint32_t s = min(a.query_start[b], a.head.num_tokens), e = min(a.query_start[b + 1], a.head.num_tokens);
        Request r;
        r.token0 = s;
        r.n = e > s ? e - s : 0;
        r.len = min(a.seq_lens[b], room);
        s_req[b] = r;
        const uint32_t rows = r.n * group;
        if (!rows) continue;
        const uint32_t top = size_for(rows);
        most = max(most, top);
        uint32_t n = 0, mid_tiles = 0, mid_cost = 0, long_tiles = 0, long_cost = 0;
#pragma unroll
        for (uint32_t i = 0; i < kSizes; ++i) {
            if (i <= top) {  // (at larger sizes the request is the same one unit)
                const uint32_t R = 32u << i;
                n = (rows + R - 1) >> (5 + i);
                const uint32_t mid = n / 2 * R, last = (n - 1) * R, per_tile = product_cost(R);
                long_tiles = unit_of(a.head, b, r, group, last, min(R, rows - last)).tile_end;
                mid_tiles = mid == last ? long_tiles : unit_of(a.head, b, r, group, mid, R).tile_end;
                long_cost = long_tiles * per_tile + item_cost(R);
                mid_cost = mid_tiles * per_tile + item_cost(R);
            }
            units_of[i] += n;
            work_of[i] += (uint64_t)n * mid_cost;
            long_of[i] = max(long_of[i], long_cost);
        }
        bytes += mid_tiles * bytes_cost(a.head.d);
        products += (uint64_t)n * mid_tiles * product_cost(32u << top);
        if (top == 0) {
            ++streams;
            streamed += mid_tiles;
            stream_long = max(stream_long, mid_tiles);
        }
    }
    if (wave * 64 < batch) {
        most = wave_scan(most, Max{});
        bytes = wave_scan(bytes, Sum{});
        products = wave_scan(products, Sum{});
        streams = wave_scan(streams, Sum{});
        streamed = wave_scan(streamed, Sum{});
        stream_long = wave_scan(stream_long, Max{});
#pragma unroll
        for (uint32_t i = 0; i < kSizes; ++i) {
            work_of[i] = wave_scan(work_of[i], Sum{});
            units_of[i] = wave_scan(units_of[i], Sum{});
            long_of[i] = wave_scan(long_of[i], Max{});
        }
    }
    if (lane == 63) {
#pragma unroll
        for (uint32_t i = 0; i < kSizes; ++i) {
            s_work[wave][i] = work_of[i];
            s_units[wave][i] = units_of[i];
            s_long[wave][i] = long_of[i];
        }
        s_most[wave] = most;
        s_bytes[wave] = bytes;
        s_products[wave] = products;
        s_streams[wave] = streams;
        s_streamed[wave] = streamed;
        s_stream_long[wave] = stream_long;
    }
    s_bucket[tid] = 0;
    __syncthreads();
    if (wave < kSizes) {  // a wave estimates a size
        const uint32_t w = lane % kPlanWaves;
        const bool own = lane < kPlanWaves;
        uint64_t work = wave_scan(own ? s_work[w][wave] : (uint64_t)0, Sum{});
        const uint32_t U = wave_scan(own ? s_units[w][wave] : 0u, Sum{});
        uint32_t longest = wave_scan(own ? s_long[w][wave] : 0u, Max{});
        most = wave_scan(s_most[w], Max{});
        bytes = wave_scan(own ? s_bytes[w] : (uint64_t)0, Sum{});
        products = wave_scan(own ? s_products[w] : (uint64_t)0, Sum{});
        streams = wave_scan(own ? s_streams[w] : 0u, Sum{});
        streamed = wave_scan(own ? s_streamed[w] : (uint64_t)0, Sum{});
        stream_long = wave_scan(s_stream_long[w], Max{});
        uint32_t per_tile = kStreamTile;
        if (bytes > products) {
            per_tile = stream_cost(a.head.d);
            work += streamed * (per_tile - kStreamTile);
            if (streams) longest = max(longest, stream_long * per_tile + item_cost(32));
        }
        streamed = streamed * per_tile + (uint64_t)streams * item_cost(32);
        const Estimate e = estimate(U, work, longest, streamed, 32u << wave, lanes);
        if (lane == 63) {
            s_time[wave] = wave > most ? ~0ull : min(e.whole, e.cut);
            if (wave == 0) {
                s_streamed[kPlanWaves] = streamed;
                s_streams[kPlanWaves] = per_tile;
            }
        }
    }
    __syncthreads();
    streamed = s_streamed[kPlanWaves];
    const uint32_t stream_tile = s_streams[kPlanWaves];
    uint32_t size = 0;
#pragma unroll
    for (uint32_t i = 1; i < kSizes; ++i)
        if (s_time[i] <= s_time[size] && s_time[i] != ~0ull) size = i;
    const uint32_t unit_rows = 32u << size;

    // The units.  Their bound holds for any ascending query_start; the clamp
    // also keeps the units of an array that is none inside the plan.
    uint32_t U = 0;
    for (uint32_t b0 = 0; b0 < batch; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        uint32_t n = 0, sum;
        if (b < batch) {
            const uint32_t rows = s_req[b].n * group;
            n = ((uint64_t)rows + unit_rows - 1) >> (5 + size);
        }
        const uint32_t at = block_scan(n, &sum);
        if (b < batch) s_first[b] = min(U + at, max_units);
        U = min(U + sum, max_units);
    }
    if (tid == 0) s_first[batch] = U;
    __syncthreads();
    uint64_t* const cost = U <= kLocalUnits ? s_cost : reinterpret_cast<uint64_t*>(base + lay.costs);
    uint64_t work = 0;
    uint32_t longest = 0;
    for (uint32_t i0 = 0; i0 < U; i0 += kPlanThreads) {
        const uint32_t i = i0 + tid;
        uint64_t c = 0, sum;
        if (i < U) {
            const uint32_t b = last_at_most(s_first, batch, i);
            const Request r = s_req[b];
            const uint32_t rows = r.n * group, row0 = (i - s_first[b]) << (5 + size);
            PagedItem u = unit_of(a.head, b, r, group, row0, min(unit_rows, rows - row0));
            const uint32_t per_tile = rows <= 32 ? stream_tile : product_cost(u.rows);
            u.next = per_tile;  // (here; the items' own below)
            units[i] = u;
            if (i < kPlanThreads) s_unit[i] = u;
            c = (uint64_t)u.tile_end * per_tile + item_cost(u.rows);
            longest = max(longest, (uint32_t)c);
        }
        const uint64_t at = block_scan(c, &sum);
        if (i < U) cost[i] = work + at;
        work += sum;
    }
    if (tid == 0) cost[U] = work;
    longest = wave_scan(longest, Max{});
    if (lane == 63) s_long[wave][0] = longest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) longest = max(longest, s_long[w][0]);

    auto unit = [&](uint32_t i) -> PagedItem { return i < kPlanThreads ? s_unit[i] : units[i]; };
    const Estimate e = estimate(U, work, longest, streamed, unit_rows, lanes);
    const uint32_t levels = e.levels;
    uint32_t n_items = U, split_blocks = 0, ranges = max(U, lanes);
    if (e.whole <= e.cut) {
        // Whole units, longest first (by cost buckets; the order within one
        // decides only which lane runs a unit, never a result).
        const float to_bucket = (float)(kBuckets - 1) / (float)max(longest, 1u);
        for (int pass = 0; pass < 2; ++pass) {
            for (uint32_t i = tid; i < U; i += kPlanThreads) {
                const uint32_t q = (uint32_t)((float)(cost[i + 1] - cost[i]) * to_bucket);
                const uint32_t bucket = kBuckets - 1 - min(kBuckets - 1, q), at = atomicAdd(&s_bucket[bucket], 1u);
                if (pass == 1) {
                    PagedItem u = unit(i);
                    u.next = kPagedNone;
                    items[at] = u;
                }
            }
            __syncthreads();
            if (pass == 0) {
                uint32_t sum;
                const uint32_t at = block_scan(s_bucket[tid], &sum);
                s_bucket[tid] = at;
                __syncthreads();
            }
        }
        if (tid < lanes && tid >= U) items[tid].rows = 0;
    } else {
        // Cut r: the start of range r, its unit and the tile in it.
        ranges = levels * lanes;
        for (uint32_t r = tid; r <= ranges; r += kPlanThreads) {
            const uint32_t level = r / lanes, nth = r % lanes;
            const uint32_t before = level >= levels ? kParts : level ? kFirstParts : 0;
            const uint32_t size = (levels == 1 || level ? kParts : kFirstParts) - before;
            const uint64_t x = work * ((uint64_t)before * lanes + (uint64_t)size * nth) / ((uint64_t)kParts * lanes);
            uint32_t i = r == ranges ? U : last_at_most(cost, U, x), t = 0;
            if (i < U) {
                const PagedItem u = unit(i);
                const uint32_t tiles = u.tile_end, per_tile = u.next, item = item_cost(u.rows);
                const uint64_t off = x - cost[i];
                if (off > item)
                    t = (uint32_t)((off - item + per_tile * kPieceTiles / 2) / (per_tile * kPieceTiles)) * kPieceTiles;
                if (t + kPieceTiles > tiles && t > 0) {
                    t = 0;
                    ++i;
                }
            }
            s_cut_unit[r] = i;
            s_cut_tile[r] = t;
        }
        __syncthreads();
        n_items = 0;
        for (uint32_t r0 = 0; r0 < ranges; r0 += kPlanThreads) {
            const uint32_t r = r0 + tid;
            uint32_t n = 0, sum;
            if (r < ranges) {
                const uint32_t u0 = s_cut_unit[r], u1 = s_cut_unit[r + 1];
                n = u1 - u0 + (s_cut_tile[r + 1] > (u0 == u1 ? s_cut_tile[r] : 0));
                if (n == 0) items[r].rows = 0;
            }
            const uint32_t at = block_scan(n, &sum);
            if (r < ranges) s_item[r] = n_items + at;
            n_items += sum;
        }
        if (tid == 0) s_item[ranges] = n_items;
        __syncthreads();
        uint32_t blocks = 0;
        for (uint32_t j0 = 0; j0 < n_items; j0 += kPlanThreads) {
            const uint32_t j = j0 + tid;
            uint32_t r = 0, i = 0, nb = 0, sum;
            PagedItem u{};
            if (j < n_items) {
                r = last_at_most(s_item, ranges, j);
                i = s_cut_unit[r] + (j - s_item[r]);
                u = unit(i);
                const uint32_t tiles = u.tile_end;
                if (j == s_item[r]) u.tile_begin = s_cut_tile[r];
                if (i == s_cut_unit[r + 1]) u.tile_end = s_cut_tile[r + 1];
                if (u.tile_begin > 0 || u.tile_end < tiles) nb = (u.rows + kPagedBlockRows - 1) / kPagedBlockRows;
                u.next = j + 1 < s_item[r + 1] ? ranges + j + 1 : kPagedNone;
            }
            const bool opens = nb && u.tile_begin == 0;
            // Two sums in one: each stays below 2^16 (paged_partial_blocks).
            const uint32_t at = block_scan(nb | (opens ? nb << 16 : 0u), &sum);
            const uint32_t first = blocks + (at & 0xffffu), sb = split_blocks + (at >> 16);
            blocks += sum & 0xffffu;
            split_blocks += sum >> 16;
            if (j < n_items) {
                if (nb) u.partial = first;
                items[j == s_item[r] ? r : ranges + j] = u;
            }
            if (opens) {
                // The range of the unit's last piece: the one before the first
                // cut past the unit.
                uint32_t lo = r, hi = ranges;
                while (hi - lo > 1) {
                    const uint32_t mid = (lo + hi) / 2;
                    if (s_cut_unit[mid] > i)
                        hi = mid;
                    else
                        lo = mid;
                }
                const uint32_t pieces = s_item[lo] + (i - s_cut_unit[lo]) - j + 1;
                for (uint32_t k = 0; k < nb; ++k) {
                    PagedSplitBlock s{};
                    s.token0 = u.token0;
                    s.row0 = u.row0 + k * kPagedBlockRows;
                    s.rows = min(kPagedBlockRows, u.rows - k * kPagedBlockRows);
                    s.first = first + k;
                    s.stride = nb;
                    s.pieces = pieces;
                    s.req = u.req;
                    s.pos0 = u.pos0;
                    split[sb + k] = s;
                }
            }
        }
    }
    if (tid == 0) {
        PagedPlanHeader& h = *reinterpret_cast<PagedPlanHeader*>(base);
        h.batch = batch;
        h.num_tokens = a.head.num_tokens;
        h.page_size = a.head.page_size;
        h.max_blocks = a.head.max_blocks;
        h.window = a.head.window;
        h.sinks = a.head.sinks;
        h.hq = a.head.hq;
        h.hkv = hkv;
        h.d = a.head.d;
        h.magic = kPagedMagic;
        h.items = n_items;
        h.split_blocks = split_blocks;
        h.ranges = ranges;
        h.units = U;
    }
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, a);
    return hipGetLastError();
}

}  // namespace tiattn
