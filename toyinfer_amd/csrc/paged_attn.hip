// Attention of new tokens over a paged KV cache, for gfx950.
//
// A persistent grid of one workgroup of eight waves per compute unit runs the
// items of a plan (paged_plan.hip): up to 256 (token, head) rows of one request
// and KV head against a range of its 64-key tiles.  Packing the query heads of
// a group into the rows lets one K/V tile serve them all, for a decoded token
// (rows = group) as for a chunk.  Four forms by the unit's rows, all of 32 rows
// per wave on v_mfma_f32_32x32x16_bf16, with the operand layouts of the prefill
// kernel (S^T = K Q^T, O^T += V^T P^T, a lane owns one row):
//   > 128 rows: eight waves of 32 rows share each tile;
//   65..128:    four waves of 32 rows share a tile, two tiles at a time;
//   33..64:     two waves of 32 rows share a 32-key half, four halves at a time;
//   <= 32:      kStreams waves stream 32-key halves of their own, without
//               barriers: K's operands go from LDS to registers, the next K is
//               requested into the place they leave, likewise V, so a wave's
//               loads are in flight while it computes.
// K and V reach LDS by buffer loads that write it.  Each instruction fills 1 KiB,
// 4 (head_dim 128) or 8 (64) rows, which lie in one page: its address is a scalar
// 64-bit base and a lane's constant.  The bases of an item's tiles, one per
// min(page size, 64) keys, wait in LDS.  Rows past the last key that the unit
// sees are some row of its last page and masked like any hidden key; V's are
// zeroed in LDS, since 0 * NaN is NaN.  Where a tile has a key that some row
// does not see and its V holds infinities or NaN, 0 times them turns that row
// to NaN: the wave marks its block of rows, and the second kernel computes the
// marked blocks again, key by key.  (Done here instead, in registers that the
// compiler took from the loops, it cost the streaming form 15 %.)  A block whose
// rows all see the value is not marked: its NaN is the result.
//
// Measured, at 32 query and 8 KV heads of 128:
//   streaming, 32 requests of 2208..8193 keys (704 MB): 114 us, 6.2 TB/s of keys
//     and values where a contiguous cache streams at 6.5; 64 KB of loads in flight per
//     compute unit is what LDS leaves beside the merge;
//   > 128 rows, a prompt of 8192: 523 to 544 us from card to card, 1.01 to 1.05 PFLOP/s;
//     matrix cores busy for 48 % of the cycles, waves waiting for 29 %.  Lanes end up to
//     6 % from their mean; the contiguous prefill attention, without pages and lists,
//     takes 480 to 494;
//   streaming at head_dim 64, half the bytes in flight: 32 such requests 66 us, 5.3 TB/s.
// What a SIMD's two waves do is in step, from barrier to barrier.  Two groups of
// waves half a tile apart, so that one multiplies while the other takes
// exponentials, took 577 us with one barrier per tile and 601 with two.
// Starting an item costs 5 us of a lane (the item, its table and queries, and
// the first keys, each waiting for the one before), ending it 1.5 to 2.5.
#include <math.h>

#include "common.hpp"
#include "paged.hpp"

namespace tiattn {
namespace {

typedef short v4i16_t __attribute__((ext_vector_type(4)));

constexpr int kPaThreads = 512;
constexpr int kPaWaves = kPaThreads / 64;
constexpr int kStreams = 4;
constexpr uint32_t kTabEntries = 1024;        // bases in LDS at a time
constexpr float kPaRescale = 8.0f;            // a running reference moves up by more than 2^8 only
constexpr float kPaMassMax = 0x1p64f, kPaMassMin = 0x1p-64f;

__device__ __forceinline__ v4i16_t read_tr16(const uint16_t* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16_t*)(p));
}

// LDS rows of D, 16-byte chunks XOR-swizzled by row (K: operand reads, V:
// transposing reads), as the prefill kernels lay theirs out.
template <int D>
__device__ __forceinline__ int pk_swz(int row) { return row & (D / 8 - 1); }
template <int D>
__device__ __forceinline__ int pv_swz(int row) { return D == 128 ? 4 * (row & 3) : 2 * (row & 3); }

template <int D>
struct PaShape {
    static constexpr int KSTEPS = D / 16;
    static constexpr int DBLK = D / 32;
    static constexpr int CPR = D / 8;            // 16-byte chunks per row
    static constexpr int RI = 64 / CPR;          // rows per load instruction
    static constexpr int HALF_LOADS = 32 / RI;   // instructions per 32 rows
    static constexpr int NF = D / 8;             // float4 per lane of a 32-row block's output
    static constexpr int TILE = 2 * 64 * D;      // elements: K and V of one tile
    static constexpr int BUF = 2 * TILE;         // of one step
};

// Where an item's keys lie (all uniform).
struct KeySource {
    const char* k;
    const char* v;
    uint64_t page_bytes;
    uint32_t row_bytes, page_shift, entry_shift, key_end;
    uint32_t low_tile, sink_tiles;
    __device__ __forceinline__ uint32_t key0(uint32_t t) const {
        return (t < sink_tiles ? t : t - sink_tiles + low_tile) * kPagedTile;
    }
};

// Lane `entry` of `bases` (byte offsets of an entry's rows in the caches).
__device__ __forceinline__ uint64_t base_of(uint2 bases, uint32_t entry) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(bases.y, entry) << 32 |
           (uint32_t)__builtin_amdgcn_readlane(bases.x, entry);
}

// (Buffer loads: the compiler counts a global load that writes LDS as an LDS
// access too and then waits for all of them before every operand.)
template <int AUX>
__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint16_t* lds) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, AUX);
}
// A resource that starts at `base`: a lane adds at most eight rows.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_at(const char* base) { return make_rsrc(base, 0x7fffffffu); }

// Rows of a wave: this lane's position; the wave's first and last, and the
// first keys inside their windows (uniform).
struct RowView {
    int32_t pos, first, last, first_low, last_low;
    uint32_t window, sinks;  // window 2^31: none
    // (Of a row before position 0, whose subtraction could wrap: key 0.)
    __device__ __forceinline__ int32_t low_of(int32_t p) const {
        return (int32_t)(max((uint32_t)(max(p, -1) + 1), window) - window);
    }
    __device__ __forceinline__ void span(int32_t f, int32_t l) {
        first = f;
        last = l;
        first_low = low_of(f);
        last_low = low_of(l);
    }
    // No row of the wave sees a key of [k0, k1].
    __device__ __forceinline__ bool none(int32_t k0, int32_t k1) const {
        return k0 > last || (k1 < first_low && (uint32_t)k0 >= sinks);
    }
    // Some row does not see some key of [k0, k1].
    __device__ __forceinline__ bool some_hidden(int32_t k0, int32_t k1) const {
        return k1 > first || (k0 < last_low && (uint32_t)k1 >= sinks);
    }
};

template <int D>
struct RowState {
    f32x16_t o[D / 32];
    float m, l;  // running reference (log2) and this lane's half of the row sum against it
};

template <int D>
__device__ __forceinline__ void clear(RowState<D>& s) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) s.o[db][i] = 0.0f;
    s.m = 0.0f;
    s.l = 0.0f;
}

// Scores to probabilities against the running reference, as the prefill
// kernel: the reference (0 at first) moves only when a probability would leave
// range or the row has next to no mass, then to the tile's maximum.  A row
// that has seen nothing yet keeps 0.
template <int D, int NB>
__device__ __forceinline__ void probabilities(f32x16_t (&st)[NB], RowState<D>& s, bf16x8_t (&pf)[2 * NB],
                                              float scale_log2) {
    auto probs = [&](float mref) __attribute__((always_inline)) {
        float sum[2 * NB];
#pragma unroll
        for (int tt = 0; tt < 2 * NB; ++tt) {
            float e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                e[j] = __builtin_amdgcn_exp2f(fmaf(st[tt / 2][8 * (tt & 1) + j], scale_log2, -mref));
            // P.V multiplies the bf16 probabilities, so the sum is taken of those.
            // (Against 64 bits the output is then off by 0.0023 of its RMS, where
            // its own rounding to bf16 alone is 0.0017.)
            const uint4 w = make_uint4(pack_bf16x2(e[0], e[1]), pack_bf16x2(e[2], e[3]), pack_bf16x2(e[4], e[5]),
                                       pack_bf16x2(e[6], e[7]));
            pf[tt] = as_bf16x8(w);
            sum[tt] = tt & 1 ? sum_bf16x8(w, sum[tt - 1]) : sum_bf16x8(w, 0.0f);
        }
        return NB == 2 ? sum[1] + sum[2 * NB - 1] : sum[1];
    };
    float ts = probs(s.m);
    const float mass = xor32_sum(s.l + ts);
    if (__any(!(ts <= kPaMassMax) || !(mass >= kPaMassMin))) {
        float mx = -INFINITY;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[nb][i]);
        const float mt = xor32_max(mx) * scale_log2;
        const bool first = xor32_sum(s.l) == 0.0f;
        if (first && mt > -INFINITY) s.m = mt;
        const bool need = !first && mt > s.m + kPaRescale;
        if (__any(need)) {
            float alpha = 1.0f;
            if (need) {
                alpha = __builtin_amdgcn_exp2f(s.m - mt);
                s.m = mt;
            }
            s.l *= alpha;
#pragma unroll
            for (int db = 0; db < D / 32; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) s.o[db][i] *= alpha;
        }
        ts = probs(s.m);
    }
    s.l += ts;
}

// Minus infinity over the scores of keys that this lane's row does not see.
template <int D, int NB>
__device__ __forceinline__ void hide(f32x16_t (&st)[NB], const RowView& rv, uint32_t k0, int kg) {
    // Keeps the branch around this: as selects it would run for every tile.
    asm volatile("; hidden keys");
    const int32_t ago = rv.pos - (int32_t)k0 - 4 * kg;  // of the lane's first key; key c of it lies ago - c behind the row
    const int32_t sinks = min((int32_t)min(rv.sinks, 0x7fffffffu), rv.pos + 1) - (int32_t)k0 - 4 * kg;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int32_t c = 32 * nb + 8 * (i / 4) + i % 4;
            const float x = c < sinks ? st[nb][i] : -INFINITY;
            st[nb][i] = (uint32_t)(ago - c) < rv.window ? st[nb][i] : x;
        }
}

// V^T operand of k-step tt (16 keys), d-block db.
template <int D>
__device__ __forceinline__ uint4 v_operand(const uint16_t* vb, int v_off, int tt) {
    const uint2 lo = __builtin_bit_cast(uint2, read_tr16(vb + v_off + 16 * tt * D));
    const uint2 hi = __builtin_bit_cast(uint2, read_tr16(vb + v_off + (16 * tt + 8) * D));
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// Both bf16 of a word all exponent bits set -> bits 7.. of each half; the
// lowest bit of each half: that half is not finite.
__device__ __forceinline__ uint32_t nonfinite_halves(uint32_t w) {
    const uint32_t e = w & 0x7f807f80u;
    return ((e & 0xffffu) == 0x7f80u ? 1u : 0u) | ((e >> 16) == 0x7f80u ? 0x10000u : 0u);
}

// Whether the 32 NB rows from vb on hold infinities or NaN.
template <int D, int NB>
__device__ __forceinline__ bool any_nonfinite(const uint16_t* vb, int lane) {
    uint32_t bad = 0;
#pragma unroll 1
    for (int i = 0; i < 32 * NB * D / 512; ++i) {
        const uint4 v = *reinterpret_cast<const uint4*>(vb + 512 * i + 8 * lane);
        bad |= nonfinite_halves(v.x) | nonfinite_halves(v.y) | nonfinite_halves(v.z) | nonfinite_halves(v.w);
    }
    return __any(bad != 0);
}

template <int D, int NB>
__device__ __forceinline__ void values(RowState<D>& s, const uint16_t* vb, const int (&v_off)[D / 32],
                                       const bf16x8_t (&pf)[2 * NB]) {
    constexpr int DBLK = D / 32;
    // Operands one k-step ahead of their products.
    uint4 va[2][DBLK];
#pragma unroll
    for (int db = 0; db < DBLK; ++db) va[0][db] = v_operand<D>(vb, v_off[db], 0);
#pragma unroll
    for (int tt = 0; tt < 2 * NB; ++tt) {
        if (tt + 1 < 2 * NB) {
#pragma unroll
            for (int db = 0; db < DBLK; ++db) va[(tt + 1) & 1][db] = v_operand<D>(vb, v_off[db], tt + 1);
        }
#pragma unroll
        for (int db = 0; db < DBLK; ++db) s.o[db] = mfma32x32x16(as_bf16x8(va[tt & 1][db]), pf[tt], s.o[db]);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 4 * DBLK, 0);
#pragma unroll
    for (int tt = 0; tt + 1 < 2 * NB; ++tt) {
        __builtin_amdgcn_sched_group_barrier(0x008, DBLK, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * DBLK, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, DBLK, 0);
}

// One tile of 32 NB keys from LDS.
template <int D, int NB>
__device__ __forceinline__ void tile(RowState<D>& s, const uint16_t* kb, const uint16_t* vb,
                                     const int (&k_off)[D / 16], const int (&v_off)[D / 32],
                                     const bf16x8_t (&qf)[D / 16], const RowView& rv, uint32_t k0, uint32_t key_end,
                                     float scale_log2, int lane, bool& bad) {
    const int kg = lane >> 5;
    constexpr int KSTEPS = D / 16;
    f32x16_t st[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i) st[nb][i] = 0.0f;
    uint4 ka[2][NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) ka[0][nb] = *reinterpret_cast<const uint4*>(kb + 32 * nb * D + k_off[0]);
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ++ks) {
        if (ks + 1 < KSTEPS) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                ka[(ks + 1) & 1][nb] = *reinterpret_cast<const uint4*>(kb + 32 * nb * D + k_off[ks + 1]);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) st[nb] = mfma32x32x16(as_bf16x8(ka[ks & 1][nb]), qf[ks], st[nb]);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * NB, 0);
#pragma unroll
    for (int ks = 0; ks + 2 < KSTEPS; ++ks) {
        __builtin_amdgcn_sched_group_barrier(0x008, NB, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, NB, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 2 * NB, 0);
    const uint32_t k1 = k0 + 32 * NB - 1;
    const bool hidden = rv.some_hidden(k0, k1);
    if (hidden) hide<D, NB>(st, rv, k0, kg);
    bf16x8_t pf[2 * NB];
    probabilities<D, NB>(st, s, pf, scale_log2);
    if (hidden && rv.some_hidden(k0, min(k1, key_end - 1)) && any_nonfinite<D, NB>(vb, lane)) bad = true;
    values<D, NB>(s, vb, v_off, pf);
}

// What the workgroup runs next, in LDS: an item or, of a streamed one, as many
// of its tiles as a table holds.
constexpr uint32_t kSegEntries = kTabEntries / 2;
struct Segment {
    PagedItem it;      // tile_end is the segment's; the item's is below
    uint32_t kvh, kind, item_end, opens;
    uint32_t token, head;  // of the unit's first row, the head in its group
    int32_t pos;
    uint32_t spoilt;       // a stream met an infinity or NaN in V of a hidden key
};

// The kernel's arguments, read again where they are used: in registers
// throughout, they would push the loops' own out.
__device__ __forceinline__ const PagedAttnArgs& arguments() {
    typedef __attribute__((address_space(4))) const PagedAttnArgs* args_t;
    args_t p = (args_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const PagedAttnArgs*)p;
}

// What every form needs of an item.
struct ItemView {
    PagedItem it;
    KeySource src;
    uint32_t kvh, group, token, head;
    int32_t pos;
    float inv_group;
};

__device__ __forceinline__ void point_at(ItemView& v, const PagedAttnArgs& a, const PagedItem& it, uint32_t kvh) {
    v.it = it;
    v.kvh = kvh;
    v.src.key_end = it.key_end;
    v.src.low_tile = it.low_tile;
    v.src.sink_tiles = it.sink_tiles;
    v.src.k = reinterpret_cast<const char*>(a.k_cache + (uint64_t)kvh * a.head.d);
    v.src.v = reinterpret_cast<const char*>(a.v_cache + (uint64_t)kvh * a.head.d);
}
__device__ __forceinline__ void point_at(ItemView& v, const PagedAttnArgs& a, const Segment& s) {
    point_at(v, a, s.it, s.kvh);
    v.token = s.token;
    v.head = s.head;
    v.pos = s.pos;
}

// Tokens that row `row` (< 256) of the unit lies behind its first row's.  The
// quotient is exact: it is at least 0.5 / group from an integer, and its error
// below 2^-22 of itself.
__device__ __forceinline__ uint32_t tokens_on(const ItemView& v, uint32_t row) {
    return (uint32_t)(((float)(v.head + row) + 0.5f) * v.inv_group);
}
// Offset of its row of q and o, in rows of D.
__device__ __forceinline__ uint64_t row_of(const PagedAttnArgs& a, const ItemView& v, uint32_t row) {
    const uint32_t t = tokens_on(v, row);
    return (uint64_t)(v.token + t) * a.head.hq + v.kvh * v.group + (v.head + row - t * v.group);
}

// The page that holds a key, and its rows' base in the caches, by the entry that
// the key lies in.  Past the last key seen: that one's.
__device__ __forceinline__ uint32_t page_of(const PagedAttnArgs& a, const ItemView& v, uint32_t key) {
    const uint32_t k = min(key, v.src.key_end - 1);
    return a.block_tables[(uint64_t)v.it.req * a.head.max_blocks + (k >> v.src.page_shift)];
}
__device__ __forceinline__ uint2 base_in(const PagedAttnArgs& a, const ItemView& v, uint32_t key, uint32_t page) {
    const uint32_t in_page = (1u << v.src.page_shift) - 1, in_entry = (1u << v.src.entry_shift) - 1;
    const uint32_t k = min(key, (v.src.key_end - 1) & ~in_entry);
    const uint64_t base = min(page, a.num_pages - 1) * v.src.page_bytes + (uint64_t)(k & in_page) * v.src.row_bytes;
    return make_uint2((uint32_t)base, (uint32_t)(base >> 32));
}
// First key of entry i of the tiles from c0 on: entry e of a tile is for its
// keys from e << entry_shift on.
__device__ __forceinline__ uint32_t entry_key(const ItemView& v, uint32_t c0, uint32_t i) {
    const uint32_t per_shift = 6 - v.src.entry_shift;
    return v.src.key0(c0 + (i >> per_shift)) + ((i & ((1u << per_shift) - 1)) << v.src.entry_shift);
}

// Q^T operand of this lane's row.
template <int D>
__device__ __forceinline__ void load_rows(bf16x8_t (&qf)[D / 16], const PagedAttnArgs& a, const ItemView& v,
                                          uint32_t row, int kg) {
    const uint16_t* q = a.q + row_of(a, v, row) * D + 8 * kg;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) qf[ks] = as_bf16x8(ldg16(q + 16 * ks));
}

// Four values of a row's output (float4 f of its fragment order): bf16 to o,
// or as they are to the item's partial results.
template <int D>
__device__ __forceinline__ void put(const PagedAttnArgs& a, const ItemView& v, uint32_t row_block, int lane, int f,
                                    float4 x, float l) {
    const uint32_t row = row_block * kPagedBlockRows + (lane & 31);
    if (row >= v.it.rows) return;
    if (v.it.partial != kPagedWhole) {
        const uint64_t blk = (uint64_t)v.kvh * paged_partial_blocks(a.head.hkv) + v.it.partial + row_block;
        reinterpret_cast<float4*>(a.part_o)[(blk * PaShape<D>::NF + f) * 64 + lane] = x;
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a row that saw nothing: 0
    uint16_t* o = a.o + row_of(a, v, row) * D + 8 * f + 4 * (lane >> 5);
    *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
}
__device__ __forceinline__ void put_ml(const PagedAttnArgs& a, const ItemView& v, uint32_t row_block, int lane,
                                       float m, float l) {
    // (The block behind the unit's last is another piece's.)
    if (v.it.partial == kPagedWhole || lane >= 32 || row_block * kPagedBlockRows >= v.it.rows) return;
    const uint64_t blk = (uint64_t)v.kvh * paged_partial_blocks(a.head.hkv) + v.it.partial + row_block;
    a.part_ml[blk * kPagedBlockRows + lane] = make_float2(m, l);
}

// By one wave: the 32-row block of the unit from `row` on is to be computed again.
__device__ __forceinline__ void mark(const PagedAttnArgs& a, const ItemView& v, uint32_t row) {
    const uint32_t t = tokens_on(v, row);
    PagedMark m{};
    m.req = v.it.req;
    m.token = v.token + t;
    m.head = v.head + row - t * v.group;
    m.kvh = v.kvh;
    m.pos = v.pos + (int32_t)t;
    m.rows = min(kPagedBlockRows, v.it.rows - row);
    if ((threadIdx.x & 63) != 0) return;
    const uint32_t n = atomicAdd(a.flags, 1u);
    if (n < kPagedMarks) a.marks[n] = m;
}

// Merge of the KS waves (streams) that hold the same 32 rows, through s_a and
// s_b, and the output.  Wave = stream * RB + row
// block; the 8 / RB waves of a row block share its output.
template <int D, int RB, int KS = kPaWaves / RB>
__device__ __forceinline__ void finish(const PagedAttnArgs& a, const ItemView& v, RowState<D>& s, uint16_t* s_a,
                                       uint16_t* s_b, float2 (*s_ml)[32], int wave, int lane) {
    constexpr int NF = PaShape<D>::NF, PARTS = kPaWaves / RB;
    const int rb = wave % RB, part = wave / RB;
    const float l = xor32_sum(s.l);
    if constexpr (KS == 1) {
        if (v.it.partial == kPagedWhole) {
            // Through LDS into rows, 16 bytes a lane: as the lanes hold them, each
            // store would touch 32 rows.
            constexpr int CPR = PaShape<D>::CPR, RI = PaShape<D>::RI;
            uint16_t* const own = (wave < 4 ? s_a : s_b) + (wave & 3) * 32 * D;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a row that saw nothing: 0
            int at = (lane & 31) * D + 8 * (lane & (CPR - 1)) + 4 * (lane >> 5);
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const float x0 = s.o[f / 4][4 * (f % 4)] * inv, x1 = s.o[f / 4][4 * (f % 4) + 1] * inv;
                const float x2 = s.o[f / 4][4 * (f % 4) + 2] * inv, x3 = s.o[f / 4][4 * (f % 4) + 3] * inv;
                *reinterpret_cast<uint2*>(own + (at ^ 8 * f)) =
                    make_uint2(pack_bf16x2(x0, x1), pack_bf16x2(x2, x3));
            }
            int ln = lane;
            asm volatile("" : "+v"(ln) : : "memory");  // (the rows' places are made after the accumulators are gone)
#pragma unroll
            for (int i = 0; i < 32 / RI; ++i) {
                const int r = RI * i + ln / CPR, c = ln % CPR;
                const uint32_t row = rb * kPagedBlockRows + r;
                const uint4 x = *reinterpret_cast<const uint4*>(own + r * D + 8 * (c ^ (r & (CPR - 1))));
                if (row < v.it.rows) *reinterpret_cast<uint4*>(a.o + row_of(a, v, row) * D + 8 * c) = x;
            }
            return;
        }
#pragma unroll
        for (int f = 0; f < NF; ++f)
            put<D>(a, v, rb, lane, f,
                   make_float4(s.o[f / 4][4 * (f % 4)], s.o[f / 4][4 * (f % 4) + 1], s.o[f / 4][4 * (f % 4) + 2],
                               s.o[f / 4][4 * (f % 4) + 3]),
                   l);
        put_ml(a, v, rb, lane, s.m, l);
        return;
    } else {
        auto area = [&](int w) __attribute__((always_inline)) {
            return reinterpret_cast<float4*>(w < 4 ? s_a : s_b) + (w & 3) * NF * 64;
        };
        __syncthreads();  // (an item without tiles comes here straight from the last one's merge)
        if (part < KS) {
            float4* const mine = area(wave);
#pragma unroll
            for (int f = 0; f < NF; ++f)
                mine[f * 64 + lane] = make_float4(s.o[f / 4][4 * (f % 4)], s.o[f / 4][4 * (f % 4) + 1],
                                                  s.o[f / 4][4 * (f % 4) + 2], s.o[f / 4][4 * (f % 4) + 3]);
            if (lane < 32) s_ml[wave][lane] = make_float2(s.m, l);
        }
        __syncthreads();
        float m = -INFINITY, w[KS], den = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const float2 ml = s_ml[k * RB + rb][lane & 31];
            w[k] = ml.x;
            if (ml.y != 0.0f) m = fmaxf(m, ml.x);
        }
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const float lk = s_ml[k * RB + rb][lane & 31].y;
            w[k] = lk != 0.0f ? __builtin_amdgcn_exp2f(w[k] - m) : 0.0f;
            den = fmaf(w[k], lk, den);
        }
#pragma unroll
        for (int i = 0; i < NF / PARTS; ++i) {
            const int f = part * (NF / PARTS) + i;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const float4 y = area(k * RB + rb)[f * 64 + lane];
                x.x = fmaf(w[k], y.x, x.x);
                x.y = fmaf(w[k], y.y, x.y);
                x.z = fmaf(w[k], y.z, x.z);
                x.w = fmaf(w[k], y.w, x.w);
            }
            put<D>(a, v, rb, lane, f, x, den);
        }
        if (part == 0) put_ml(a, v, rb, lane, m == -INFINITY ? 0.0f : m, den);
    }
}

// Workgroup barrier that waits for this wave's LDS operations only and leaves
// its loads in flight.
__device__ __forceinline__ void lds_ops_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// More than 32 rows: RB = 8, 4 or 2 row blocks.  A step is one tile (RB = 8) or
// two, filled by all waves; stream s of the 8 / RB takes its own 64 (RB >= 4) or
// 32 keys of it.
template <int D, int RB>
__device__ __forceinline__ void run_shared(const PagedAttnArgs& a, const ItemView& v, uint16_t* s_a, uint16_t* s_b,
                                           uint2* s_tab, float2 (*s_ml)[32], float scale_log2, RowView rv) {
    using P = PaShape<D>;
    constexpr int KS = kPaWaves / RB, TILES = RB == 8 ? 1 : 2, NB = 2 * TILES / KS;
    constexpr int ROWS = 64 * TILES / kPaWaves, LOADS = ROWS / P::RI;  // per wave, step and tensor
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 31, kg = lane >> 5, rb = wave % RB, stream = wave / RB;
    const uint32_t per_shift = 6 - v.src.entry_shift, chunk = kTabEntries >> per_shift;

    // A wave loads ROWS consecutive rows of the step, RI per instruction; this
    // lane's bytes of an instruction's rows.
    const int lr = lane / P::CPR, phys = lane % P::CPR;
    const int fill_tile = ROWS * wave / 64, fill_row = ROWS * wave % 64;
    uint32_t koff[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
        koff[j] = ((P::RI * j & 7) + lr) * v.src.row_bytes + 16 * (phys ^ pk_swz<D>(fill_row + P::RI * j + lr));
    uint32_t voff[8 / P::RI];
#pragma unroll
    for (int j = 0; j < 8 / P::RI; ++j) voff[j] = (P::RI * j + lr) * v.src.row_bytes + 16 * (phys ^ pv_swz<D>(lr));
    int k_off[P::KSTEPS], v_off[P::DBLK];
#pragma unroll
    for (int ks = 0; ks < P::KSTEPS; ++ks) k_off[ks] = ql * D + 8 * ((2 * ks + kg) ^ pk_swz<D>(ql));
    {
        const int s16 = lane & 15, g16 = lane >> 4, vrow = 4 * kg + (s16 >> 2);
#pragma unroll
        for (int db = 0; db < P::DBLK; ++db)
            v_off[db] = vrow * D + 8 * ((4 * db + 2 * (g16 & 1) + ((s16 & 3) >> 1)) ^ pv_swz<D>(vrow)) + 4 * (s16 & 1);
    }
    const uint32_t last_row = v.it.rows - 1, row = min((uint32_t)(rb * 32 + ql), last_row);
    const uint32_t w_first = min((uint32_t)rb * 32, last_row), w_last = min((uint32_t)rb * 32 + 31, last_row);
    rv.pos = v.pos + (int32_t)tokens_on(v, row);
    rv.span(v.pos + (int32_t)__builtin_amdgcn_readfirstlane(tokens_on(v, w_first)),
            v.pos + (int32_t)__builtin_amdgcn_readfirstlane(tokens_on(v, w_last)));
    const bool live = rb * 32 < (int)v.it.rows;
    bf16x8_t qf[P::KSTEPS];
    load_rows<D>(qf, a, v, row, kg);
    RowState<D> s;
    clear(s);
    bool bad = false;

    for (uint32_t c0 = v.it.tile_begin; c0 < v.it.tile_end; c0 += chunk) {
        const uint32_t c1 = min(v.it.tile_end, c0 + chunk);
        // The first step's loads wait for their own table entries only, not for
        // the whole table.
        constexpr int OWN = kTabEntries / kPaThreads;
        const uint32_t n = (c1 - c0) << per_shift;
        const uint32_t own_key = entry_key(v, min(c0 + fill_tile, c1 - 1) , lane & ((1u << per_shift) - 1));
        const uint32_t own_page = page_of(a, v, own_key);
        uint32_t page[OWN];
#pragma unroll
        for (int u = 0; u < OWN; ++u) {
            const uint32_t i = threadIdx.x + u * kPaThreads;
            page[u] = i < n ? page_of(a, v, entry_key(v, c0, i)) : 0;
        }
        // This wave's part of the step from tile t on (its tile may lie past the
        // last).
        auto bases_of = [&](uint32_t t) __attribute__((always_inline)) {
            return s_tab[((min(t + fill_tile, c1 - 1) - c0) << per_shift) + (lane & ((1u << per_shift) - 1))];
        };
        auto fill = [&](uint32_t t, uint2 bases, uint16_t* buf) __attribute__((always_inline)) {
            if (TILES > 1 && t + fill_tile >= c1) return;
            uint16_t* const to = buf + P::TILE * fill_tile;
#pragma unroll
            for (int g = 0; g < ROWS / 8; ++g) {  // eight rows: one page
                const uint32_t r = fill_row + 8 * g;
                const uint64_t off = base_of(bases, r >> v.src.entry_shift) +
                                     (r & ((1u << v.src.entry_shift) - 1)) * v.src.row_bytes;
                const __amdgpu_buffer_rsrc_t rk = rows_at(v.src.k + off), rv = rows_at(v.src.v + off);
#pragma unroll
                for (int i = 0; i < 8 / P::RI; ++i) {
                    load_lds16<0>(rk, koff[g * (8 / P::RI) + i], to + D * (r + P::RI * i));
                    load_lds16<0>(rv, voff[i], to + D * (64 + r + P::RI * i));
                }
            }
        };
        // This wave's loads of the step from tile t into buf, and zeros over its
        // rows of V past the last key seen.  The wait is explicit: the compiler's
        // tracking of loads that write LDS is not relied on.
        auto land = [&](uint32_t t, uint16_t* buf) __attribute__((always_inline)) {
            __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
            const uint32_t k0 = v.src.key0(t + fill_tile) + fill_row;
            if (t + fill_tile < c1 && k0 + ROWS > v.src.key_end) {
#pragma unroll
                for (int j = 0; j < LOADS; ++j)
                    if (k0 + P::RI * j + lr >= v.src.key_end)
                        *reinterpret_cast<uint4*>(buf + P::TILE * fill_tile + D * (64 + fill_row + P::RI * j) + 8 * lane) =
                            make_uint4(0, 0, 0, 0);
            }
            __syncthreads();
        };
        lds_ops_barrier();  // the table's and the tiles' last readers are done
        fill(c0, base_in(a, v, own_key, own_page), s_a);
#pragma unroll
        for (int u = 0; u < OWN; ++u) {
            const uint32_t i = threadIdx.x + u * kPaThreads;
            if (i < n) s_tab[i] = base_in(a, v, entry_key(v, c0, i), page[u]);
        }
        lds_ops_barrier();
        uint2 bases = bases_of(c0 + TILES);
        land(c0, s_a);
        // The step from tile t out of `cur` while the next streams into `nxt`,
        // whose last readers passed the previous barrier.
        constexpr int KEYS = 32 * NB;
        const int my_tile = KEYS * stream / 64, my_row = KEYS * stream % 64;
        auto step = [&](uint32_t t, const uint16_t* cur, uint16_t* nxt) __attribute__((always_inline)) {
            if (t + TILES < c1) {
                fill(t + TILES, bases, nxt);
                bases = bases_of(t + 2 * TILES);
            }
            const uint32_t k0 = v.src.key0(t + my_tile) + my_row;
            const uint16_t* const kb = cur + P::TILE * my_tile + D * my_row;
            if (live && (TILES == 1 || t + my_tile < c1) && !rv.none(k0, k0 + KEYS - 1))
                tile<D, NB>(s, kb, kb + 64 * D, k_off, v_off, qf, rv, k0, v.src.key_end, scale_log2, lane, bad);
            land(t + TILES, nxt);
        };
        for (uint32_t t = c0; t < c1; t += 2 * TILES) {
            step(t, s_a, s_b);
            if (t + TILES < c1) step(t + TILES, s_b, s_a);
        }
    }
    if (bad) mark(arguments(), v, rb * 32);
    finish<D, RB, KS>(arguments(), v, s, s_a, s_b, s_ml, wave, lane);
}

// Operand reads of the streaming form, in asm: to the compiler they are no LDS
// accesses, which it would make wait for every load in flight that writes LDS.
// Each block waits for its own reads.  The swizzles make a k-step's (K) or a
// d-block's (V) address the first one's with a bit or two flipped.
template <int KSTEPS>
__device__ __forceinline__ void read_k(uint4 (&k)[KSTEPS], uint2& bases, uint32_t at, uint32_t bases_at) {
    typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
    typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
    u4_t r[KSTEPS];
    u2_t e;
    if constexpr (KSTEPS == 8)
        asm volatile(
            "ds_read_b64 %8, %17\n\t"
            "ds_read_b128 %0, %9\n\t"
            "ds_read_b128 %1, %10\n\t"
            "ds_read_b128 %2, %11\n\t"
            "ds_read_b128 %3, %12\n\t"
            "ds_read_b128 %4, %13\n\t"
            "ds_read_b128 %5, %14\n\t"
            "ds_read_b128 %6, %15\n\t"
            "ds_read_b128 %7, %16\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]),
              "=&v"(e)
            : "v"(at), "v"(at ^ 32), "v"(at ^ 64), "v"(at ^ 96), "v"(at ^ 128), "v"(at ^ 160), "v"(at ^ 192),
              "v"(at ^ 224), "v"(bases_at)
            : "memory");
    else
        asm volatile(
            "ds_read_b64 %4, %9\n\t"
            "ds_read_b128 %0, %5\n\t"
            "ds_read_b128 %1, %6\n\t"
            "ds_read_b128 %2, %7\n\t"
            "ds_read_b128 %3, %8\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(e)
            : "v"(at), "v"(at ^ 32), "v"(at ^ 64), "v"(at ^ 96), "v"(bases_at)
            : "memory");
#pragma unroll
    for (int i = 0; i < KSTEPS; ++i) k[i] = make_uint4(r[i].x, r[i].y, r[i].z, r[i].w);
    bases = make_uint2(e.x, e.y);
}

// V^T operands of 32 keys: v[tt][db].
__device__ __forceinline__ void read_v(uint4 (&v)[2][4], uint32_t at) {
    typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
    u2_t r[16];  // d-block 0: keys 0, 8, 16, 24 on; d-block 1: ...
    asm volatile(
        "ds_read_b64_tr_b16 %0, %16\n\t"
        "ds_read_b64_tr_b16 %1, %16 offset:2048\n\t"
        "ds_read_b64_tr_b16 %2, %16 offset:4096\n\t"
        "ds_read_b64_tr_b16 %3, %16 offset:6144\n\t"
        "ds_read_b64_tr_b16 %4, %17\n\t"
        "ds_read_b64_tr_b16 %5, %17 offset:2048\n\t"
        "ds_read_b64_tr_b16 %6, %17 offset:4096\n\t"
        "ds_read_b64_tr_b16 %7, %17 offset:6144\n\t"
        "ds_read_b64_tr_b16 %8, %18\n\t"
        "ds_read_b64_tr_b16 %9, %18 offset:2048\n\t"
        "ds_read_b64_tr_b16 %10, %18 offset:4096\n\t"
        "ds_read_b64_tr_b16 %11, %18 offset:6144\n\t"
        "ds_read_b64_tr_b16 %12, %19\n\t"
        "ds_read_b64_tr_b16 %13, %19 offset:2048\n\t"
        "ds_read_b64_tr_b16 %14, %19 offset:4096\n\t"
        "ds_read_b64_tr_b16 %15, %19 offset:6144\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7]),
          "=&v"(r[8]), "=&v"(r[9]), "=&v"(r[10]), "=&v"(r[11]), "=&v"(r[12]), "=&v"(r[13]), "=&v"(r[14]), "=&v"(r[15])
        : "v"(at), "v"(at ^ 64), "v"(at ^ 128), "v"(at ^ 192)
        : "memory");
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int db = 0; db < 4; ++db)
            v[tt][db] = make_uint4(r[4 * db + 2 * tt].x, r[4 * db + 2 * tt].y, r[4 * db + 2 * tt + 1].x,
                                   r[4 * db + 2 * tt + 1].y);
}
__device__ __forceinline__ void read_v(uint4 (&v)[2][2], uint32_t at) {
    typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
    u2_t r[8];
    constexpr int kRows8 = 8 * 64 * 2;  // bytes of eight rows
    asm volatile(
        "ds_read_b64_tr_b16 %0, %8\n\t"
        "ds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
        "ds_read_b64_tr_b16 %2, %8 offset:%11\n\t"
        "ds_read_b64_tr_b16 %3, %8 offset:%12\n\t"
        "ds_read_b64_tr_b16 %4, %9\n\t"
        "ds_read_b64_tr_b16 %5, %9 offset:%10\n\t"
        "ds_read_b64_tr_b16 %6, %9 offset:%11\n\t"
        "ds_read_b64_tr_b16 %7, %9 offset:%12\n\t"
        "s_waitcnt lgkmcnt(0)"
        : "=&v"(r[0]), "=&v"(r[1]), "=&v"(r[2]), "=&v"(r[3]), "=&v"(r[4]), "=&v"(r[5]), "=&v"(r[6]), "=&v"(r[7])
        : "v"(at), "v"(at ^ 64), "n"(kRows8), "n"(2 * kRows8), "n"(3 * kRows8)
        : "memory");
#pragma unroll
    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int db = 0; db < 2; ++db)
            v[tt][db] = make_uint4(r[4 * db + 2 * tt].x, r[4 * db + 2 * tt].y, r[4 * db + 2 * tt + 1].x,
                                   r[4 * db + 2 * tt + 1].y);
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return (uint32_t)(size_t)(const __attribute__((address_space(3))) void*)p;
}

// A plan entry that no launch in flight writes, by scalar loads.
template <typename T>
__device__ __forceinline__ T plan_load(const void* plan, uint64_t byte) {
    static_assert(sizeof(T) % 16 == 0, "whole loads");
    typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
    u4_t w[sizeof(T) / 16];
#pragma unroll
    for (size_t i = 0; i < sizeof(T) / 16; ++i)
        w[i] = reinterpret_cast<const u4_t __attribute__((address_space(4)))*>(
            (uint64_t)plan + byte)[i];
    return __builtin_bit_cast(T, w);
}

// The part of the header that the kernels read.  A plan that was made for
// other arguments does not fit: the attention then fills o with NaN.
struct PlanHead {
    uint32_t batch, num_tokens, page_size, max_blocks, window, sinks, hq, hkv, d, magic, items, split_blocks, ranges, units;
    uint32_t pad[2];
    __device__ __forceinline__ bool fits(const PagedPlanHeader& w) const {
        return ((batch ^ w.batch) | (num_tokens ^ w.num_tokens) | (page_size ^ w.page_size) |
                (max_blocks ^ w.max_blocks) | (window ^ w.window) | (sinks ^ w.sinks) | (hq ^ w.hq) | (hkv ^ w.hkv) |
                (d ^ w.d) | (magic ^ kPagedMagic)) == 0;
    }
};

enum : uint32_t { kSegNone = 0, kSegStream = 1, kSegShared = 2 };

// By one wave: `it` of KV head `kvh` from tile `from` on as a segment, with the
// table and the query rows of a streamed one.
template <int D>
__device__ __forceinline__ void stage(const PagedAttnArgs& a, ItemView& v, PagedItem it, uint32_t kvh, uint32_t from,
                                      Segment* seg, uint2* tab, uint16_t* q) {
    const uint32_t lane = threadIdx.x & 63;
    const bool opens = from == it.tile_begin;
    const uint32_t item_end = it.tile_end, ahead = it.row0 / v.group;
    point_at(v, a, it, kvh);
    v.token = it.token0 + ahead;
    v.head = it.row0 - ahead * v.group;
    v.pos = it.pos0 + (int32_t)ahead;
    uint32_t kind = kSegShared;
    if (it.rows <= 32) {
        kind = kSegStream;
        const uint32_t per_shift = 6 - v.src.entry_shift;
        it.tile_begin = from;
        it.tile_end = min(item_end, from + (kSegEntries >> per_shift));
        if (opens) {
            constexpr uint32_t CPR = D / 8;
            for (uint32_t i = lane; i < it.rows * CPR; i += 64) {
                const uint32_t row = i / CPR, c = i % CPR;
                *reinterpret_cast<uint4*>(q + row * D + 8 * (c ^ pk_swz<D>(row))) =
                    ldg16(a.q + row_of(a, v, row) * D + 8 * c);
            }
        }
        for (uint32_t i = lane; i < (it.tile_end - it.tile_begin) << per_shift; i += 64) {
            const uint32_t key = entry_key(v, it.tile_begin, i);
            tab[i] = base_in(a, v, key, page_of(a, v, key));
        }
    }
    if (lane == 0) {
        Segment s;
        s.it = it;
        s.kvh = kvh;
        s.kind = kind;
        s.item_end = item_end;
        s.opens = opens;
        s.token = v.token;
        s.head = v.head;
        s.pos = v.pos;
        s.spoilt = 0;
        *seg = s;
    }
}

// By one wave: what follows item `it` of KV head `kvh` in its list, or the
// list of a ticket (`drawn`: lane 0 holds one), staged.
template <int D>
__device__ __forceinline__ void advance(const PagedAttnArgs& a, ItemView& v, const PlanHead& head, PagedItem it,
                                        uint32_t kvh, bool drawn, uint32_t ticket, Segment* seg, uint2* tab,
                                        uint16_t* q) {
    const uint32_t lane = threadIdx.x & 63, hkv = a.head.hkv, lanes = paged_lanes(hkv);
    uint32_t idx = it.next;
    while (true) {
        if (idx == kPagedNone) {
            if (head.ranges <= lanes) break;
            if (!drawn && lane == 0) ticket = atomicAdd(a.tickets + kvh, 1u);
            drawn = false;
            idx = lanes + __builtin_amdgcn_readfirstlane(ticket);
            // This head's lists are gone: the head with the most left.  The
            // counters only grow, so this ends.
            while (idx >= head.ranges) {
                const uint32_t mine = (kvh + lane) % hkv;
                const uint32_t gone = __hip_atomic_load(a.tickets + mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                uint32_t least = gone;
#pragma unroll
                for (int m = 32; m >= 1; m >>= 1) least = min(least, (uint32_t)__shfl_xor(least, m));
                if (lanes + least >= head.ranges) break;
                kvh = __builtin_amdgcn_readlane(mine, __builtin_ctzll(__ballot(gone == least)));
                if (lane == 0) ticket = atomicAdd(a.tickets + kvh, 1u);
                idx = lanes + __builtin_amdgcn_readfirstlane(ticket);
            }
            if (idx >= head.ranges) break;
        }
        it = plan_load<PagedItem>(a.plan, sizeof(PagedPlanHeader) + (uint64_t)idx * sizeof(PagedItem));
        if (it.rows) {
            stage<D>(a, v, it, kvh, it.tile_begin, seg, tab, q);
            return;
        }
        idx = kPagedNone;  // an empty list
    }
    if (lane == 0) seg->kind = kSegNone;
}

// Up to 32 rows: wave w < kStreams streams the 32-key halves w, w + kStreams,
// ... of a segment's tiles, and on into the next segment, which wave kStreams
// stages meanwhile: a wave's first loads of it go out behind its last ones of
// this, and are in flight while the streams merge.  (Staged by all waves after
// the merge, a new item cost 20 us of its workgroup under load: its ticket, the
// item, the table and the first keys are fetched one after the other.)
// Runs segments from `slot` on; returns the slot of one that is not streamed.
template <int D>
__device__ __forceinline__ uint32_t run_streams(const PagedAttnArgs& a, ItemView v, const PlanHead& head,
                                                uint32_t slot, Segment* s_seg, uint16_t* s_a, uint16_t* s_b,
                                                uint2* s_tab, uint16_t* s_q, float2 (*s_ml)[32], float scale_log2,
                                                RowView rv) {
    using P = PaShape<D>;
    constexpr int NL = P::HALF_LOADS, NF = P::NF, NT = 2;  // non-temporal: the keys are read once
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 31, kg = lane >> 5;
    const uint32_t per_shift = 6 - v.src.entry_shift, half = wave & 1;
    uint16_t* const sk = s_a + (wave % kStreams) * 32 * D;
    uint16_t* const sv = s_b + (wave % kStreams) * 32 * D;
    // The merge lies behind the streams' tiles: stream k's 32 rows in fragment
    // order at merge_at(k).
    const uint32_t merge_a = lds_address(s_a + P::BUF / 2), merge_b = lds_address(s_b + P::BUF / 2);
    static_assert(kStreams * 32 * D <= P::BUF / 2 && kStreams == 4, "tiles in the first half, two streams' rows in each second");
    auto merge_at = [&](int k) __attribute__((always_inline)) {
        return (k < 2 ? merge_a : merge_b) + (k & 1) * NF * 1024 + 16 * lane;
    };

    const int lr = lane / P::CPR, phys = lane % P::CPR;
    constexpr int SWZ = D / 8 / P::RI;  // instructions after which K's swizzle repeats
    uint32_t koff[SWZ];
#pragma unroll
    for (int j = 0; j < SWZ; ++j)
        koff[j] = ((P::RI * j & 7) + lr) * v.src.row_bytes + 16 * (phys ^ pk_swz<D>(P::RI * j + lr));
    uint32_t voff[8 / P::RI];
#pragma unroll
    for (int j = 0; j < 8 / P::RI; ++j) voff[j] = (P::RI * j + lr) * v.src.row_bytes + 16 * (phys ^ pv_swz<D>(lr));
    int v_off[P::DBLK];
    {
        const int s16 = lane & 15, g16 = lane >> 4, vrow = 4 * kg + (s16 >> 2);
#pragma unroll
        for (int db = 0; db < P::DBLK; ++db)
            v_off[db] = vrow * D + 8 * ((4 * db + 2 * (g16 & 1) + ((s16 & 3) >> 1)) ^ pv_swz<D>(vrow)) + 4 * (s16 & 1);
    }
    const uint32_t k_at = lds_address(sk + ql * D + 8 * (kg ^ pk_swz<D>(ql))), v_at = lds_address(sv + v_off[0]);
    // This wave's halves lie in one half of their tiles.
    auto fill_k = [&](const char* from, uint2 bases) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {  // eight rows: one page
            const uint32_t r = 32 * half + 8 * g;
            const __amdgpu_buffer_rsrc_t rows = rows_at(from + base_of(bases, r >> v.src.entry_shift) +
                                                        (r & ((1u << v.src.entry_shift) - 1)) * v.src.row_bytes);
#pragma unroll
            for (int i = 0; i < 8 / P::RI; ++i)
                load_lds16<NT>(rows, koff[(g * (8 / P::RI) + i) % SWZ], sk + D * (8 * g + P::RI * i));
        }
    };
    auto fill_v = [&](const char* from, uint2 bases) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const uint32_t r = 32 * half + 8 * g;
            const __amdgpu_buffer_rsrc_t rows = rows_at(from + base_of(bases, r >> v.src.entry_shift) +
                                                        (r & ((1u << v.src.entry_shift) - 1)) * v.src.row_bytes);
#pragma unroll
            for (int i = 0; i < 8 / P::RI; ++i) load_lds16<NT>(rows, voff[i], sv + D * (8 * g + P::RI * i));
        }
    };
    // Entry of half h of a segment that begins at tile c0.
    auto entry_of = [&](uint32_t at, uint32_t h, uint32_t c0) __attribute__((always_inline)) {
        return s_tab + at * kSegEntries + (((h >> 1) - c0) << per_shift) + (lane & ((1u << per_shift) - 1));
    };
    // Of a segment: the halves that hold a key which is seen end here.
    auto end_of = [&](const PagedItem& it) __attribute__((always_inline)) {
        if (it.tile_end <= it.tile_begin) return 2 * it.tile_begin;
        KeySource k = v.src;
        k.low_tile = it.low_tile;
        k.sink_tiles = it.sink_tiles;
        return k.key0(it.tile_end - 1) + 32 < it.key_end ? 2 * it.tile_end : 2 * it.tile_end - 1;
    };
    auto segment = [&](uint32_t at) __attribute__((always_inline)) {
        Segment s;
        uint32_t w[sizeof(Segment) / 4];
#pragma unroll
        for (size_t i = 0; i < sizeof(Segment) / 4; ++i)
            w[i] = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t*>(s_seg + at)[i]);
        __builtin_memcpy(&s, w, sizeof(s));
        return s;
    };

    // All waves, after the streams' results are in LDS.
    auto merge = [&]() __attribute__((always_inline)) {
        float m = -INFINITY, w[kStreams], den = 0.0f;
#pragma unroll
        for (int k = 0; k < kStreams; ++k) {
            const float2 ml = s_ml[k][lane & 31];
            w[k] = ml.x;
            if (ml.y != 0.0f) m = fmaxf(m, ml.x);
        }
#pragma unroll
        for (int k = 0; k < kStreams; ++k) {
            const float lk = s_ml[k][lane & 31].y;
            w[k] = lk != 0.0f ? __builtin_amdgcn_exp2f(w[k] - m) : 0.0f;
            den = fmaf(w[k], lk, den);
        }
#pragma unroll
        for (int i = 0; i < NF / kPaWaves; ++i) {
            const int f = wave * (NF / kPaWaves) + i;
            f32x4_t y[kStreams];
            asm volatile(
                "ds_read_b128 %0, %4\n\t"
                "ds_read_b128 %1, %5\n\t"
                "ds_read_b128 %2, %6\n\t"
                "ds_read_b128 %3, %7\n\t"
                "s_waitcnt lgkmcnt(0)"
                : "=&v"(y[0]), "=&v"(y[1]), "=&v"(y[2]), "=&v"(y[3])
                : "v"(merge_at(0) + f * 1024), "v"(merge_at(1) + f * 1024), "v"(merge_at(2) + f * 1024),
                  "v"(merge_at(3) + f * 1024)
                : "memory");
            f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < kStreams; ++k) x += w[k] * y[k];
            put<D>(a, v, 0, lane, f, make_float4(x.x, x.y, x.z, x.w), den);
        }
        if (wave == 0) put_ml(a, v, 0, lane, m == -INFINITY ? 0.0f : m, den);
    };

    if (wave >= kStreams) {
        while (true) {
            const Segment seg = segment(slot);
            if (seg.kind != kSegStream) return slot;
            point_at(v, a, seg);
            const bool closes = seg.it.tile_end == seg.item_end;
            if (wave == kStreams) {
                const uint32_t to = slot ^ 1;
                PagedItem it = seg.it;
                it.tile_end = seg.item_end;
                ItemView w = v;
                if (closes)
                    advance<D>(a, w, head, it, seg.kvh, false, 0, s_seg + to, s_tab + to * kSegEntries, s_q + to * 32 * D);
                else
                    stage<D>(a, w, it, seg.kvh, seg.it.tile_end, s_seg + to, s_tab + to * kSegEntries, s_q + to * 32 * D);
            }
            lds_ops_barrier();  // the next segment is staged
            lds_ops_barrier();  // this one's results are in LDS, its table and rows done with
            if (closes) merge();
            if (wave == kStreams && s_seg[slot].spoilt) mark(a, v, 0);
            slot ^= 1;
        }
    }
    RowState<D> s;
    bf16x8_t qf[P::KSTEPS];
    bool armed = false;  // this wave's first loads of the segment are out
    while (true) {
        const Segment seg = segment(slot);
        if (seg.kind != kSegStream) return slot;
        point_at(v, a, seg);
        const bool closes = seg.it.tile_end == seg.item_end;
        bool next_has = false;
        const uint32_t last_row = seg.it.rows - 1, row = min((uint32_t)ql, last_row);
        rv.pos = v.pos + (int32_t)tokens_on(v, row);
        rv.span(v.pos, v.pos + (int32_t)__builtin_amdgcn_readfirstlane(tokens_on(v, last_row)));
        const uint32_t c0 = seg.it.tile_begin, end = end_of(seg.it);
        uint32_t h = 2 * c0 + wave;
        const uint32_t n = h < end ? (end - h + kStreams - 1) / kStreams : 0;
        if (!armed && n) {
            const uint2 bases = *entry_of(slot, h, c0);
            fill_k(v.src.k, bases);
            fill_v(v.src.v, bases);
        }
        if (seg.opens) {
            const uint16_t* const q = s_q + slot * 32 * D + row * D;
#pragma unroll
            for (int ks = 0; ks < P::KSTEPS; ++ks)
                qf[ks] = as_bf16x8(*reinterpret_cast<const uint4*>(q + 8 * ((2 * ks + kg) ^ pk_swz<D>(row))));
            clear(s);
        }
        // The next segment is known from this iteration on.
        const uint32_t meet = n > 2 ? 2 : n ? n - 1 : 0;
        const char *next_k = nullptr, *next_v = nullptr;
        uint32_t next_c0 = 0;
        auto look_ahead = [&]() __attribute__((always_inline)) {
            lds_ops_barrier();
            const Segment nx = segment(slot ^ 1);
            if (nx.kind != kSegStream) return;
            next_c0 = nx.it.tile_begin;
            next_has = 2 * next_c0 + wave < end_of(nx.it);
            next_k = reinterpret_cast<const char*>(a.k_cache + (uint64_t)nx.kvh * D);
            next_v = reinterpret_cast<const char*>(a.v_cache + (uint64_t)nx.kvh * D);
        };
        if (n == 0) {
            look_ahead();
            if (next_has) {
                const uint2 bases = *entry_of(slot ^ 1, 2 * next_c0 + wave, next_c0);
                fill_k(next_k, bases);
                fill_v(next_v, bases);
            }
        }
        for (uint32_t i = 0; i < n; ++i, h += kStreams) {
            if (i == meet) look_ahead();
            const uint32_t k0 = v.src.key0(h >> 1) + 32 * half;
            const bool inside = i + 1 < n, more = inside || next_has;
            const char* const from_k = inside ? v.src.k : next_k;
            const char* const from_v = inside ? v.src.v : next_v;
            const uint2* const entry = inside     ? entry_of(slot, h + kStreams, c0)
                                       : next_has ? entry_of(slot ^ 1, 2 * next_c0 + wave, next_c0)
                                                  : entry_of(slot, h, c0);
            // K has landed (V, requested after it, may not have): its operands
            // to registers, then the next K into its place.
            __builtin_amdgcn_s_waitcnt(wait_vmcnt(NL));
            uint4 ka[P::KSTEPS];
            uint2 bases;
            read_k(ka, bases, k_at, lds_address(entry));
            if (more) fill_k(from_k, bases);
            f32x16_t st[1];
#pragma unroll
            for (int j = 0; j < 16; ++j) st[0][j] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < P::KSTEPS; ++ks) st[0] = mfma32x32x16(as_bf16x8(ka[ks]), qf[ks], st[0]);
            const uint32_t k1 = k0 + 31;
            const bool hidden = rv.some_hidden(k0, k1);
            if (hidden) hide<D, 1>(st, rv, k0, kg);
            bf16x8_t pf[2];
            probabilities<D, 1>(st, s, pf, scale_log2);
            // V likewise: of what is in flight only the next K came after it.
            if (more)
                __builtin_amdgcn_s_waitcnt(wait_vmcnt(NL));
            else
                __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
            if (hidden) {
                asm volatile("" ::: "memory");
#pragma unroll
                for (int j = 0; j < NL; ++j)
                    if (k0 + P::RI * j + lr >= v.src.key_end)
                        *reinterpret_cast<uint4*>(sv + 512 * j + 8 * lane) = make_uint4(0, 0, 0, 0);
                __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
                if (rv.some_hidden(k0, min(k1, v.src.key_end - 1)) && any_nonfinite<D, 1>(sv, lane)) s_seg[slot].spoilt = 1;
            }
            uint4 va[2][P::DBLK];
            read_v(va, v_at);
            if (more) fill_v(from_v, bases);
#pragma unroll
            for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                for (int db = 0; db < P::DBLK; ++db)
                    s.o[db] = mfma32x32x16(as_bf16x8(va[tt][db]), pf[tt], s.o[db]);
        }
        if (closes) {
            const float l = xor32_sum(s.l);
            const uint32_t to = merge_at(wave);
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const f32x4_t x = {s.o[f / 4][4 * (f % 4)], s.o[f / 4][4 * (f % 4) + 1], s.o[f / 4][4 * (f % 4) + 2],
                                   s.o[f / 4][4 * (f % 4) + 3]};
                asm volatile("ds_write_b128 %0, %1 offset:%2" ::"v"(to), "v"(x), "n"(f * 1024) : "memory");
            }
            if (lane < 32) s_ml[wave][lane] = make_float2(s.m, l);
        }
        lds_ops_barrier();
        if (closes) merge();
        armed = next_has;
        slot ^= 1;
    }
}

template <int D>
__global__ __launch_bounds__(kPaThreads, 1) void paged_attn_kernel(PagedAttnArgs a, float scale_log2) {
    __shared__ __align__(1024) uint16_t s_a[PaShape<D>::BUF];
    __shared__ __align__(1024) uint16_t s_b[PaShape<D>::BUF];
    __shared__ uint2 s_tab[kTabEntries];
    __shared__ __align__(16) uint16_t s_q[2 * 32 * D];
    __shared__ float2 s_ml[kPaWaves][32];
    __shared__ Segment s_seg[2];
    const uint32_t hkv = a.head.hkv, lanes = paged_lanes(hkv);
    const uint32_t kvh = blockIdx.x % hkv, l = blockIdx.x / hkv;
    const PlanHead head = plan_load<PlanHead>(a.plan, 0);
    const PagedItem first = plan_load<PagedItem>(a.plan, sizeof(PagedPlanHeader) + (uint64_t)l * sizeof(PagedItem));
    if (!head.fits(a.head)) {
        const uint64_t n = (uint64_t)a.head.num_tokens * a.head.hq * (D / 8);
        for (uint64_t i = (uint64_t)blockIdx.x * kPaThreads + threadIdx.x; i < n; i += (uint64_t)gridDim.x * kPaThreads)
            reinterpret_cast<uint4*>(a.o)[i] = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
        return;
    }
    RowView rv{};
    rv.window = a.head.window && a.head.window < 0x80000000u ? a.head.window : 0x80000000u;
    rv.sinks = a.head.window ? a.head.sinks : 0;
    ItemView v{};
    v.group = a.head.hq / hkv;
    v.inv_group = 1.0f / (float)v.group;
    v.src.page_shift = 31 - __builtin_clz(a.head.page_size);
    v.src.entry_shift = min(v.src.page_shift, 6u);
    v.src.row_bytes = hkv * D * 2;
    v.src.page_bytes = 2 * a.page_stride;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t slot = 0;
    if (wave == 0) {
        ItemView w = v;
        if (first.rows)
            stage<D>(a, w, first, kvh, first.tile_begin, s_seg, s_tab, s_q);
        else  // (an empty list: further ones may not be)
            advance<D>(a, w, head, PagedItem{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, kPagedNone}, kvh, false, 0, s_seg, s_tab, s_q);
    }
    __syncthreads();
    while (s_seg[slot].kind != kSegNone) {
        if (s_seg[slot].kind == kSegStream) {
            slot = run_streams<D>(arguments(), v, head, slot, s_seg, s_a, s_b, s_tab, s_q, s_ml, scale_log2, rv);
            continue;
        }
        Segment seg;
        {
            uint32_t w[sizeof(Segment) / 4];
#pragma unroll
            for (size_t i = 0; i < sizeof(Segment) / 4; ++i)
                w[i] = __builtin_amdgcn_readfirstlane(reinterpret_cast<const uint32_t*>(s_seg + slot)[i]);
            __builtin_memcpy(&seg, w, sizeof(seg));
        }
        point_at(v, a, seg);
        // A ticket for the list after this one, drawn now and looked at below.
        const bool draws = head.ranges > lanes && seg.it.next == kPagedNone;
        uint32_t ticket = 0;
        if (draws && threadIdx.x == 0) ticket = atomicAdd(a.tickets + seg.kvh, 1u);
        if (v.it.rows > 128)
            run_shared<D, 8>(arguments(), v, s_a, s_b, s_tab, s_ml, scale_log2, rv);
        else if (v.it.rows > 64)
            run_shared<D, 4>(arguments(), v, s_a, s_b, s_tab, s_ml, scale_log2, rv);
        else
            run_shared<D, 2>(arguments(), v, s_a, s_b, s_tab, s_ml, scale_log2, rv);
        lds_ops_barrier();  // every wave is done with the tiles (its stores may still be under way)
        if (wave == 0) {
            ItemView w = v;
            advance<D>(arguments(), w, head, seg.it, seg.kvh, draws, ticket, s_seg, s_tab, s_q);
        }
        slot = 0;
        lds_ops_barrier();
    }
}

// One row's attention again, by a workgroup, key by key over those that it sees:
// a wave takes every fourth tile of 64 keys, the newest first, a lane a key for
// the scores and then D / 64 of the dims.  For rows of marked blocks only.  A row
// that the keys it sees make NaN throughout stops there.  Bound by the latency of
// its loads, 23 us per 64 keys and wave.  One NaN in V, in us: a decode batch at
// the edge of a window of 4096 keys 51 -> 570, 512 tokens on 8192 keys 89 -> 1541,
// a prompt of 8192 583 -> 716 (key 819) and 1892 (key 7372); sixteen V rows in
// flight instead of eight took up to 1.8 times that.
struct ExactLds {
    float4 q[2][16];  // even dims, odd dims
    float o[4][128];
    float2 ml[4];
    uint32_t stop;
};
static_assert(sizeof(ExactLds) <= 16384, "in the merge's LDS");
template <int D>
__device__ __forceinline__ void exact_row(const PagedAttnArgs& a, float scale_log2, uint32_t req, int32_t pos,
                                          uint32_t token, uint32_t kvh, uint32_t head, ExactLds& lds) {
    constexpr int DPL = D / 64, U = 8;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t page_shift = 31 - __builtin_clz(a.head.page_size);
    const uint32_t window = a.head.window, sinks = window ? a.head.sinks : 0;
    const uint32_t low = window && pos >= 0 && (uint32_t)pos + 1 > window ? (uint32_t)pos + 1 - window : 0;
    const uint32_t* const table = a.block_tables + (uint64_t)req * a.head.max_blocks;
    const uint64_t row = ((uint64_t)token * a.head.hq + head) * D;
    __syncthreads();  // the last row's results are read
    if (threadIdx.x == 0) lds.stop = 0;
    if (threadIdx.x < D) reinterpret_cast<float*>(lds.q[threadIdx.x & 1])[threadIdx.x / 2] = bf16_to_f32(a.q[row + threadIdx.x]);
    __syncthreads();
    float m = -INFINITY, l = 0.0f, acc[DPL];
#pragma unroll
    for (int e = 0; e < DPL; ++e) acc[e] = 0.0f;
    for (int32_t t = pos < 0 ? -1 : (pos >> 6) - (int32_t)wave; t >= 0; t -= 4) {
        if (*(volatile uint32_t*)&lds.stop) break;
        const uint32_t key = 64 * (uint32_t)t + lane;
        const bool seen = key <= (uint32_t)pos && (key >= low || key < sinks);
        const uint64_t mask = __ballot(seen);
        if (!mask) continue;
        float sc = -INFINITY;
        uint64_t at = 0;
        if (seen) {
            const uint32_t page = min(table[key >> page_shift], a.num_pages - 1);
            at = page * a.page_stride + ((uint64_t)(key & (a.head.page_size - 1)) * a.head.hkv + kvh) * D;
            float dot[2] = {0.0f, 0.0f};
#pragma unroll 8
            for (int c = 0; c < D / 8; ++c) {
                const uint4 k4 = ldg16(a.k_cache + at + 8 * c);
                const float4 q0 = lds.q[0][c], q1 = lds.q[1][c];
                dot[0] = fmaf(q0.x, bf16_lo(k4.x), fmaf(q0.y, bf16_lo(k4.y), dot[0]));
                dot[0] = fmaf(q0.z, bf16_lo(k4.z), fmaf(q0.w, bf16_lo(k4.w), dot[0]));
                dot[1] = fmaf(q1.x, bf16_hi(k4.x), fmaf(q1.y, bf16_hi(k4.y), dot[1]));
                dot[1] = fmaf(q1.z, bf16_hi(k4.z), fmaf(q1.w, bf16_hi(k4.w), dot[1]));
            }
            sc = (dot[0] + dot[1]) * scale_log2;
        }
        float mx = sc;
#pragma unroll
        for (int b = 32; b >= 1; b >>= 1) mx = fmaxf(mx, __shfl_xor(mx, b));
        if (mx > m) {
            const float alpha = __builtin_amdgcn_exp2f(m - mx);
            l *= alpha;
#pragma unroll
            for (int e = 0; e < DPL; ++e) acc[e] *= alpha;
            m = mx;
        }
        const float p = seen ? __builtin_amdgcn_exp2f(sc - (m == -INFINITY ? 0.0f : m)) : 0.0f;
        for (uint64_t left = mask; left;) {
            int j[U];
            bool has[U];
            float v[U][DPL];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                has[u] = left != 0;
                j[u] = has[u] ? __builtin_ctzll(left) : j[0];
                left &= left - 1;
                const uint16_t* const src =
                    a.v_cache + base_of(make_uint2((uint32_t)at, (uint32_t)(at >> 32)), j[u]) + DPL * lane;
                if constexpr (DPL == 2) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(src);
                    v[u][0] = bf16_lo(w);
                    v[u][1] = bf16_hi(w);
                } else {
                    v[u][0] = bf16_to_f32(*src);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (!has[u]) break;
                const float pj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), j[u]));
                l += pj;
#pragma unroll
                for (int e = 0; e < DPL; ++e) acc[e] = fmaf(pj, v[u][e], acc[e]);
            }
        }
        bool nan = l != l;
        if (!nan) {
            nan = acc[0] != acc[0];
            if constexpr (DPL == 2) nan = nan && acc[1] != acc[1];
        }
        if (__all(nan)) {
            if (lane == 0) *(volatile uint32_t*)&lds.stop = 1;
            break;
        }
    }
#pragma unroll
    for (int e = 0; e < DPL; ++e) lds.o[wave][DPL * lane + e] = acc[e];
    if (lane == 0) lds.ml[wave] = make_float2(m, l);
    __syncthreads();
    if (threadIdx.x >= D) return;
    float M = -INFINITY, x = 0.0f, tot = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) M = fmaxf(M, lds.ml[k].x);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float2 ml = lds.ml[k];
        const float w = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - M);  // (0 keeps the NaN of a sum)
        tot = fmaf(w, ml.y, tot);
        x = fmaf(w, lds.o[k][threadIdx.x], x);
    }
    a.o[row + threadIdx.x] = f32_to_bf16(x * (tot == 0.0f ? 0.0f : 1.0f / tot));
}

// Merge of the pieces of each split 32-row block: a workgroup takes one d-block
// of one row block, its waves every fourth piece, and the four partial merges
// meet in LDS.  Bound by latency: a launch with nothing to merge takes 4 to 5 us
// under a trace, 512 tokens on 8192 keys (64 blocks per head, 33 MB) 11.6 with 512
// workgroups; with as many as fit at a time the call is 2 us shorter.
constexpr uint32_t kMergeWgs = 1024;
constexpr int kMergeThreads = 256;

template <int D>
__global__ __launch_bounds__(kMergeThreads) void paged_merge_kernel(PagedAttnArgs a, float scale_log2) {
    constexpr int DBLK = D / 32, NF = PaShape<D>::NF, U = 4;
    __shared__ float4 s_o[4][4][64];
    __shared__ float2 s_ml[4][64];
    __shared__ int s_found[4];
    const PlanHead head = plan_load<PlanHead>(a.plan, 0);
    if (!head.fits(a.head)) return;
    const uint32_t hkv = a.head.hkv, group = a.head.hq / hkv, blocks = head.split_blocks;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t met = scalar_load(a.flags), marks = min(met, kPagedMarks);
    const bool all_marked = met > kPagedMarks;
    // Whether one of the first n marks names this block; the same answer to all threads.
    auto marked = [&](uint32_t n, uint32_t req, uint32_t token, uint32_t h, uint32_t kvh) {
        bool is = false;
        for (uint32_t i = threadIdx.x; i < n; i += kMergeThreads) {
            const PagedMark m = arguments().marks[i];
            is |= m.req == req && m.token == token && m.head == h && m.kvh == kvh;
        }
        const int any = __any(is);
        __syncthreads();  // (the last answer is read)
        if (lane == 0) s_found[wave] = any;
        __syncthreads();
        return (s_found[0] | s_found[1] | s_found[2] | s_found[3]) != 0;
    };
    // The tickets back to zero, for the next call.
    for (uint32_t i = blockIdx.x * kMergeThreads + threadIdx.x; i < hkv; i += kMergeWgs * kMergeThreads) a.tickets[i] = 0;
    const PagedPlanLayout lay = paged_plan_layout(a.head.batch, a.head.num_tokens, a.head.hq, hkv);
    for (uint32_t i = blockIdx.x; i < blocks * hkv * DBLK; i += kMergeWgs) {
        const uint32_t db = i % DBLK, kvh = i / DBLK % hkv;
        const PagedSplitBlock sb =
            plan_load<PagedSplitBlock>(a.plan, lay.split_blocks + (uint64_t)(i / (DBLK * hkv)) * sizeof(PagedSplitBlock));
        const uint64_t b0 = (uint64_t)kvh * paged_partial_blocks(hkv) + sb.first;
        const bool has = (uint32_t)(lane & 31) < sb.rows;
        // The place of this lane's row in o, found while the loads below are on
        // their way.
        const uint32_t r = sb.row0 + (lane & 31), token = sb.token0 + r / group, h = kvh * group + r % group;
        uint64_t at = ((uint64_t)token * a.head.hq + h) * D + 32 * db + 8 * wave + 4 * (lane >> 5);
        asm volatile("" : "+v"(at));
        float M = -INFINITY, den = 0.0f;
        float4 acc[4];
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[f] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (has) {
            for (uint32_t p0 = wave; p0 < sb.pieces; p0 += 4 * U) {
                float2 ml[U];
                float4 x[U][4];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t p = p0 + 4 * u < sb.pieces ? p0 + 4 * u : p0;
                    const uint64_t blk = b0 + (uint64_t)p * sb.stride;
                    ml[u] = a.part_ml[blk * kPagedBlockRows + (lane & 31)];
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                        x[u][f] = reinterpret_cast<const float4*>(a.part_o)[(blk * NF + 4 * db + f) * 64 + lane];
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (p0 + 4 * u >= sb.pieces || ml[u].y == 0.0f) continue;  // no such piece, or it saw nothing
                    const float Mn = fmaxf(M, ml[u].x);
                    const float wa = M == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(M - Mn);
                    const float wb = __builtin_amdgcn_exp2f(ml[u].x - Mn);
                    den = fmaf(wb, ml[u].y, wa * den);
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        acc[f].x = fmaf(wb, x[u][f].x, wa * acc[f].x);
                        acc[f].y = fmaf(wb, x[u][f].y, wa * acc[f].y);
                        acc[f].z = fmaf(wb, x[u][f].z, wa * acc[f].z);
                        acc[f].w = fmaf(wb, x[u][f].w, wa * acc[f].w);
                    }
                    M = Mn;
                }
            }
        }
        __syncthreads();  // the last round's reads are done
#pragma unroll
        for (int f = 0; f < 4; ++f) s_o[wave][f][lane] = acc[f];
        s_ml[wave][lane] = make_float2(M, den);
        __syncthreads();
        float Mt = -INFINITY, w[4], tot = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) Mt = fmaxf(Mt, s_ml[k][lane].x);
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 ml = s_ml[k][lane];
            w[k] = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - Mt);
            tot = fmaf(w[k], ml.y, tot);
            const float4 y = s_o[k][wave][lane];
            x.x = fmaf(w[k], y.x, x.x);
            x.y = fmaf(w[k], y.y, x.y);
            x.z = fmaf(w[k], y.z, x.z);
            x.w = fmaf(w[k], y.w, x.w);
        }
        const float inv = tot == 0.0f ? 0.0f : 1.0f / tot;
        // (Marked blocks are written below only.)
        if (met && (all_marked || marked(marks, sb.req, sb.token0 + sb.row0 / group, sb.row0 % group, kvh))) continue;
        if (has)
            *reinterpret_cast<uint2*>(a.o + at) =
                make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
    }
    if (!met) return;
    // The rows of the marked blocks, each block by its first mark.
    const uint64_t rows = all_marked ? (uint64_t)head.units * hkv * kPagedMaxRows : (uint64_t)marks * kPagedBlockRows;
    for (uint64_t i = blockIdx.x; i < rows; i += kMergeWgs) {
        uint32_t req, token, h, kvh, row;
        int32_t pos;
        if (all_marked) {
            const uint64_t at = i / kPagedMaxRows;
            const PagedItem u = plan_load<PagedItem>(a.plan, lay.units + at / hkv * sizeof(PagedItem));
            row = u.row0 + (uint32_t)(i % kPagedMaxRows);
            if (i % kPagedMaxRows >= u.rows) continue;
            req = u.req;
            token = u.token0;
            h = 0;
            kvh = (uint32_t)(at % hkv);
            pos = u.pos0;
        } else {
            const uint32_t at = (uint32_t)(i / kPagedBlockRows);
            const PagedMark m = plan_load<PagedMark>(arguments().marks, at * sizeof(PagedMark));
            row = i % kPagedBlockRows;
            if (row >= m.rows || marked(at, m.req, m.token, m.head, m.kvh)) continue;
            req = m.req;
            token = m.token;
            h = m.head;
            kvh = m.kvh;
            pos = m.pos;
        }
        const uint32_t ahead = (h + row) / group;
        exact_row<D>(arguments(), scale_log2, req, pos + (int32_t)ahead, token + ahead, kvh, kvh * group + (h + row) % group,
                     *reinterpret_cast<ExactLds*>(s_o));
    }
    // The count back to zero, by the last workgroup to come here (flags[1] counts them).
    __syncthreads();
    if (threadIdx.x == 0 && atomicAdd(a.flags + 1, 1u) == kMergeWgs - 1) {
        a.flags[0] = 0;
        a.flags[1] = 0;
    }
}

template <int D>
hipError_t launch_attn_t(const PagedAttnArgs& a, hipStream_t st) {
    const uint32_t wgs = a.head.hkv * paged_lanes(a.head.hkv);
    const float scale_log2 = kLog2e / sqrtf((float)D);
    hipLaunchKernelGGL((paged_attn_kernel<D>), dim3(wgs), dim3(kPaThreads), 0, st, a, scale_log2);
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL((paged_merge_kernel<D>), dim3(kMergeWgs), dim3(kMergeThreads), 0, st, a, scale_log2);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
    return a.head.d == 64 ? launch_attn_t<64>(a, stream) : launch_attn_t<128>(a, stream);
}

}  // namespace tiattn
