// Host-side launch interface of the paged-cache operators, and the layout of
// the attention plan that paged_plan.hip writes and paged_attn.hip reads.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace tiattn {

constexpr uint32_t kPagedMaxBatch = 4096;
constexpr uint32_t kNoSlot = 0xffffffffu;

// The 8-bit cache: a page is its codes [Hkv][page_size][D], one byte each, then
// the scales [Hkv][page_size / kFp8Block] in fp32.  (By head, so that a head's
// rows of a page lie in one piece and a row of 64 dims shares its line with its
// neighbours, not with other heads.)
constexpr uint32_t kFp8Block = 16;
constexpr int kFp8Low = -100, kFp8High = 119;  // exponents of the scales
inline __host__ __device__ uint64_t fp8_page_bytes(uint32_t page_size, uint32_t hkv, uint32_t d) {
    const uint64_t blocks = (uint64_t)hkv * (page_size / kFp8Block);
    return (blocks * (kFp8Block * d + sizeof(float)) + 15) / 16 * 16;
}

// ------------------------------------------------------------------ tables
struct PagedTablesArgs {
    const uint32_t* context_lens;
    const uint32_t* new_lens;
    uint32_t batch;
    const uint32_t* free_pages;
    uint32_t free_capacity;
    const uint32_t* num_free;
    uint32_t page_shift;
    uint32_t* block_tables;
    uint32_t max_blocks;
    uint32_t num_tokens;
    uint32_t* query_start;
    uint32_t* seq_lens;
    uint32_t* positions;
    uint32_t* slots;
    uint32_t* status;
};
hipError_t launch_paged_tables(const PagedTablesArgs& a, hipStream_t stream);

// ---------------------------------------------------------------- prologue
struct PagedPrologueArgs {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t* q_weight;
    const uint16_t* k_weight;
    const float* rope;
    uint32_t num_positions;
    const uint32_t* positions;
    const uint32_t* slots;
    uint32_t num_tokens;
    float eps;
    uint16_t* q_out;
    uint16_t* k_cache;
    uint16_t* v_cache;
    uint32_t num_slots;    // pages * page size
    uint32_t page_shift;
    uint64_t page_stride;  // elements
    uint32_t hq, hkv;
};
hipError_t launch_paged_prologue(const PagedPrologueArgs& a, uint32_t d, hipStream_t stream);

struct PagedPrologueFp8Args {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t* q_weight;
    const uint16_t* k_weight;
    const float* rope;
    uint32_t num_positions;
    const uint32_t* positions;
    const uint32_t* slots;
    uint32_t num_tokens;
    float eps;
    uint16_t* q_out;
    uint8_t* k_cache;
    uint8_t* v_cache;
    uint32_t num_slots;
    uint32_t page_shift;
    uint64_t page_bytes;  // from one page to the next
    uint32_t hq, hkv;
};
hipError_t launch_paged_prologue_fp8(const PagedPrologueFp8Args& a, uint32_t d, hipStream_t stream);

// -------------------------------------------------------------------- read
struct PagedReadFp8Args {
    const uint8_t* k_cache;
    const uint8_t* v_cache;
    const uint32_t* block_tables;
    const uint32_t* query_start;
    const uint32_t* seq_lens;
    uint32_t batch, num_tokens;
    uint16_t* k_out;
    uint16_t* v_out;
    uint32_t num_pages;
    uint32_t page_shift;
    uint64_t page_bytes;
    uint32_t max_blocks, hkv;
};
hipError_t launch_paged_read_fp8(const PagedReadFp8Args& a, uint32_t d, hipStream_t stream);

// --------------------------------------------------------------- attention
//
// The rows of a request, for one KV head, are (new token, query head of the
// group) pairs: row r is token r / group, head r % group.  A unit is up to 256
// consecutive rows of a request, an item a range of a unit's key tiles; the
// same units and items serve every KV head.
constexpr uint32_t kPagedTile = 64;       // keys per tile
constexpr uint32_t kPagedSlots = 256;     // workgroups: one per compute unit
constexpr uint32_t kPagedMaxRows = 256;   // rows of a unit
constexpr uint32_t kPagedBlockRows = 32;  // rows of a wave

// Lanes per KV head: workgroups that start on it.
inline __host__ __device__ uint32_t paged_lanes(uint32_t hkv) {
    return hkv >= kPagedSlots ? 1 : kPagedSlots / hkv;
}
// A plan of cut units has up to kPagedLevels ranges per lane, one with units of
// 256 rows.  A cut leaves two pieces of its unit, so per KV head the workspace
// holds this many 32-row blocks of partial results, and the plan half as many
// blocks that are in pieces.
constexpr uint32_t kPagedLevels = 2;
inline __host__ __device__ uint32_t paged_partial_blocks(uint32_t hkv) {
    return 2 * (kPagedMaxRows / kPagedBlockRows) * paged_lanes(hkv);
}

struct PagedPlanHeader {
    // The arguments that the plan was made for; the attention compares them.
    uint32_t batch, num_tokens, page_size, max_blocks, window, sinks, hq, hkv, d, magic;
    uint32_t items;
    uint32_t split_blocks;  // 32-row blocks whose partials are to be merged, per KV head
    uint32_t ranges;        // lists of items: lane l runs list l, then draws further ones
    uint32_t units;         // in the plan's array of them
    uint32_t pad[50];
};
static_assert(sizeof(PagedPlanHeader) == 256, "the items follow at a cache line");
constexpr uint32_t kPagedMagic = 0x70616765u;

constexpr uint32_t kPagedWhole = 0xffffffffu, kPagedNone = 0xffffffffu;
// Item r < ranges is the first of list r (rows 0: the list is empty).
struct PagedItem {
    uint32_t req;      // row of the block table
    uint32_t token0;   // row of q and o that holds the request's first new token
    uint32_t row0;     // first row of the unit
    uint32_t rows;     // 1..256
    int32_t pos0;      // position of the request's first new token (< 0: it sees nothing)
    uint32_t key_end;  // keys at or past it are seen by no row of the unit
    uint32_t low_tile; // tiles [0, sink_tiles) and from low_tile on are seen
    uint32_t sink_tiles;
    uint32_t tile_begin, tile_end;  // of the unit's tiles, counted through that gap
    uint32_t partial;  // first 32-row block of its partial results, or kPagedWhole
    uint32_t next;     // the list's next item, or kPagedNone
};
static_assert(sizeof(PagedItem) == 48, "read by 16-byte loads");

// One 32-row block of a split unit: its rows, and its partial blocks
// first, first + stride, ... (pieces of them).
struct PagedSplitBlock {
    uint32_t token0, row0, rows;  // as in PagedItem, of this block (rows 1..32)
    uint32_t first, stride, pieces;
    uint32_t req;
    int32_t pos0;  // as in PagedItem
};
static_assert(sizeof(PagedSplitBlock) == 32, "read by 16-byte loads");

// A 32-row block one of whose tiles had an infinity or NaN in V of a key that
// some row of the block does not see.  A workspace holds this many; if a call
// meets more (of pieces and streams each its own), all of its rows count as such.
constexpr uint32_t kPagedMarks = 4096;
struct PagedMark {
    uint32_t req;          // row of the block table
    uint32_t token, head;  // of its first row: row of q and o, head in the group
    uint32_t kvh;
    int32_t pos;
    uint32_t rows;  // 1..32
    uint32_t pad[2];
};
static_assert(sizeof(PagedMark) == 32, "read by 16-byte loads");

// Units of any plan for these sizes, and the places of the plan's arrays.
inline __host__ __device__ uint32_t paged_max_units(uint32_t batch, uint32_t num_tokens, uint32_t group) {
    return batch + (uint32_t)(((uint64_t)num_tokens * group) / kPagedBlockRows);
}
struct PagedPlanLayout {
    size_t items, split_blocks, units, costs, bytes;
};
inline __host__ __device__ PagedPlanLayout paged_plan_layout(uint32_t batch, uint32_t num_tokens,
                                                             uint32_t hq, uint32_t hkv) {
    const size_t units = paged_max_units(batch, num_tokens, hq / hkv), cuts = kPagedLevels * paged_lanes(hkv);
    PagedPlanLayout l;
    l.items = sizeof(PagedPlanHeader);
    // The ranges' first items, then at most one per unit and cut.
    l.split_blocks = l.items + (units + 2 * cuts) * sizeof(PagedItem);
    l.units = l.split_blocks + paged_partial_blocks(hkv) / 2 * sizeof(PagedSplitBlock);
    l.costs = l.units + units * sizeof(PagedItem);
    l.bytes = (l.costs + (units + 1) * sizeof(uint64_t) + 255) / 256 * 256;
    return l;
}

struct PagedPlanArgs {
    const uint32_t* query_start;
    const uint32_t* seq_lens;
    PagedPlanHeader head;  // the arguments' part
    void* plan;
};
hipError_t launch_paged_plan(const PagedPlanArgs& a, hipStream_t stream);

struct PagedAttnArgs {
    const uint16_t* q;
    const void* k_cache;
    const void* v_cache;
    uint16_t* o;
    const uint32_t* block_tables;
    const void* plan;
    PagedPlanHeader head;  // what the plan has to have been made for
    uint32_t num_pages;
    uint64_t page_bytes;   // from one page to the next
    uint32_t* tickets;     // [KV head], zero between calls
    uint32_t* flags;       // [2], zero between calls: marks; workgroups of the merge that are done
    PagedMark* marks;      // [kPagedMarks]
    float* part_o;         // [KV head][block][D / 4][64 lanes][4]
    float2* part_ml;       // [KV head][block][32 rows]: reference (log2), sum
};
hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream);
hipError_t launch_paged_attention_fp8(const PagedAttnArgs& a, hipStream_t stream);

}  // namespace tiattn
