// Attention of new tokens over a paged KV cache, for gfx950.
//
// A persistent grid of two workgroups per compute unit runs the items of a
// plan (paged_plan.hip): up to 128 (token, head) rows of one request and KV
// head against a range of its 64-key tiles.  Packing the query heads of a group
// into the rows lets one K/V tile serve them all, for a decoded token (rows =
// group) as for a chunk.  Three forms by the unit's rows, all of 32 rows per
// wave on v_mfma_f32_32x32x16_bf16, with the operand layouts of the prefill
// kernel (S^T = K Q^T, O^T += V^T P^T, a lane owns one row):
//   > 64 rows: four waves of 32 rows share each tile;
//   33..64:    two waves of 32 rows, each over one 32-key half of a tile, twice;
//   <= 32:     every wave streams 32-key halves of its own, without barriers:
//              K's operands go from LDS to registers, the next K is requested
//              into the place they leave, likewise V, so a wave's loads are in
//              flight while it computes.
// K and V reach LDS by buffer loads that write it.  Each instruction fills 1 KiB,
// 4 (head_dim 128) or 8 (64) rows, which one page holds: its buffer resource is
// built from the page's number by scalar instructions, in 64 bits, and ends
// behind the last key that the unit sees, so that rows past it read as zeros.
// The page numbers of an item wait in LDS.
#include <math.h>

#include "common.hpp"
#include "paged.hpp"

namespace tiattn {
namespace {

typedef short v4i16_t __attribute__((ext_vector_type(4)));

constexpr int kPaThreads = 256;
constexpr uint32_t kTabEntries = 2048;        // page numbers in LDS at a time
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
    static constexpr int BUF = 2 * 64 * D;       // elements: K and V of one tile
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

// RI rows from key `key` of the page that lane `entry` of `pages` names.
template <int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const KeySource& s, const char* base, uint32_t pages,
                                                           uint32_t entry, uint32_t key) {
    const uint32_t page = __builtin_amdgcn_readlane(pages, entry);
    const uint32_t in_page = key & ((1u << s.page_shift) - 1);
    const uint32_t rows = key < s.key_end ? min(s.key_end - key, (uint32_t)PaShape<D>::RI) : 0;
    const uint32_t bytes = rows ? (rows - 1) * s.row_bytes + D * 2 : 0;
    return make_rsrc(base + (uint64_t)page * s.page_bytes + (uint64_t)in_page * s.row_bytes, bytes);
}

__device__ __forceinline__ void load_lds16(__amdgpu_buffer_rsrc_t r, uint16_t* lds, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}

// Rows of a wave: this lane's position and the wave's first and last.
struct RowView {
    int32_t pos, first, last;
    uint32_t window, sinks;  // window 2^31: none
    __device__ __forceinline__ bool sees(uint32_t key) const {
        return (uint32_t)(pos - (int32_t)key) < window || ((int32_t)key <= pos && key < sinks);
    }
    // No row of the wave sees a key of [k0, k1].
    __device__ __forceinline__ bool none(uint32_t k0, uint32_t k1) const {
        return (int32_t)k0 > last || (k0 >= sinks && (int64_t)k1 + window <= (int64_t)first);
    }
    // Some row does not see some key of [k0, k1].
    __device__ __forceinline__ bool some_hidden(uint32_t k0, uint32_t k1) const {
        return (int32_t)k1 > first || ((int64_t)k0 + window <= (int64_t)last && k1 >= sinks);
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

template <int D, int NB>
__device__ __forceinline__ void hide(f32x16_t (&st)[NB], const RowView& rv, uint32_t k0, int kg) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (!rv.sees(k0 + 32 * nb + 8 * (i / 4) + 4 * kg + i % 4)) st[nb][i] = -INFINITY;
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

template <int D, int NB>
__device__ __forceinline__ bool any_nonfinite(const uint16_t* vb, const int (&v_off)[D / 32]) {
    uint32_t bad = 0;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int tt = 0; tt < 2 * NB; ++tt) {
            if (tt == 0) __builtin_amdgcn_sched_barrier(0);
            const uint4 v = v_operand<D>(vb, v_off[db], tt);
#pragma unroll
            for (int e = 0; e < 4; ++e) bad |= nonfinite_halves(word_of(v, e));
        }
    return __any(bad != 0);
}

// A word of two bf16 with those that are not finite replaced by 0.
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
    const uint32_t bad = nonfinite_halves(w);
    return w & ~(((bad & 1u) ? 0xffffu : 0u) | ((bad >> 16) ? 0xffff0000u : 0u));
}

// O^T += V^T P^T for a tile where some row does not see some key and V holds
// infinities or NaN: 0 * NaN would carry them into rows that do not see
// them.  The finite part of V multiplies P; what is not finite is added, key by
// key, to the rows that see the key.
template <int D, int NB>
__device__ __forceinline__ void values_isolated(RowState<D>& s, const uint16_t* vb, const int (&v_off)[D / 32],
                                                const bf16x8_t (&pf)[2 * NB], const RowView& rv, uint32_t k0, int kg) {
#pragma unroll
    for (int tt = 0; tt < 2 * NB; ++tt)
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
            __builtin_amdgcn_sched_barrier(0);  // one operand at a time: few registers
            uint4 v = v_operand<D>(vb, v_off[db], tt);
            v = make_uint4(finite_part(v.x), finite_part(v.y), finite_part(v.z), finite_part(v.w));
            s.o[db] = mfma32x32x16(as_bf16x8(v), pf[tt], s.o[db]);
        }
#pragma unroll 1
    for (int key = 0; key < 32 * NB; ++key) {
        const bool seen = rv.sees(k0 + key);
#pragma unroll
        for (int f = 0; f < D / 8; ++f) {
            __builtin_amdgcn_sched_barrier(0);
            const uint2 w = *reinterpret_cast<const uint2*>(vb + key * D + 8 * (f ^ pv_swz<D>(key)) + 4 * kg);
            const uint32_t x[2] = {w.x & ~finite_part(w.x), w.y & ~finite_part(w.y)};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y = e & 1 ? bf16_hi(x[e / 2]) : bf16_lo(x[e / 2]);
                s.o[f / 4][4 * (f % 4) + e] += seen ? y : 0.0f;
            }
        }
    }
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
                                     float scale_log2, int kg) {
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
    if (hidden && rv.some_hidden(k0, min(k1, key_end - 1)) && any_nonfinite<D, NB>(vb, v_off))
        values_isolated<D, NB>(s, vb, v_off, pf, rv, k0, kg);
    else
        values<D, NB>(s, vb, v_off, pf);
}

// What every form needs of an item.
struct ItemView {
    PagedItem it;
    KeySource src;
    uint32_t kvh, group;
    const uint32_t* table;   // the request's row
    uint32_t num_pages;
};

// The page numbers of tiles [c0, c1), one per min(page size, 64) keys; keys
// that no row sees get page 0 (their rows are never loaded).
__device__ __forceinline__ void fill_table(const ItemView& v, uint32_t* s_tab, uint32_t c0, uint32_t c1) {
    const uint32_t per_shift = 6 - v.src.entry_shift, n = (c1 - c0) << per_shift;
    for (uint32_t i = threadIdx.x; i < n; i += kPaThreads) {
        const uint32_t key = v.src.key0(c0 + (i >> per_shift)) + ((i & ((1u << per_shift) - 1)) << v.src.entry_shift);
        s_tab[i] = key < v.src.key_end ? min(v.table[key >> v.src.page_shift], v.num_pages - 1) : 0;
    }
}

// Q^T operand of this lane's row.
template <int D>
__device__ __forceinline__ void load_rows(bf16x8_t (&qf)[D / 16], const PagedAttnArgs& a, const ItemView& v,
                                          uint32_t row, int kg) {
    const uint32_t r = v.it.row0 + row, token = v.it.token0 + r / v.group, head = v.kvh * v.group + r % v.group;
    const uint16_t* q = a.q + ((uint64_t)token * a.head.hq + head) * D + 8 * kg;
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
    const uint32_t r = v.it.row0 + row, token = v.it.token0 + r / v.group, head = v.kvh * v.group + r % v.group;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a row that saw nothing: 0
    uint16_t* o = a.o + ((uint64_t)token * a.head.hq + head) * D + 8 * f + 4 * (lane >> 5);
    *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
}
__device__ __forceinline__ void put_ml(const PagedAttnArgs& a, const ItemView& v, uint32_t row_block, int lane,
                                       float m, float l) {
    if (v.it.partial == kPagedWhole || lane >= 32) return;
    const uint64_t blk = (uint64_t)v.kvh * paged_partial_blocks(a.head.hkv) + v.it.partial + row_block;
    a.part_ml[blk * kPagedBlockRows + lane] = make_float2(m, l);
}

// Merge of the KS waves (streams) that hold the same 32 rows, through s_a and
// s_b (free: a barrier has passed), and the output; wave = stream * (4 / KS) +
// row block.
template <int D, int KS>
__device__ __forceinline__ void finish(const PagedAttnArgs& a, const ItemView& v, RowState<D>& s, uint16_t* s_a,
                                       uint16_t* s_b, float2 (*s_ml)[32], int wave, int lane) {
    constexpr int NF = PaShape<D>::NF, RB = 4 / KS;
    const int rb = wave % RB, stream = wave / RB;
    const float l = xor32_sum(s.l);
    if constexpr (KS == 1) {
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
            return reinterpret_cast<float4*>(w < 2 ? s_a : s_b) + (w & 1) * NF * 64;
        };
        float4* const mine = area(wave);
#pragma unroll
        for (int f = 0; f < NF; ++f)
            mine[f * 64 + lane] = make_float4(s.o[f / 4][4 * (f % 4)], s.o[f / 4][4 * (f % 4) + 1],
                                              s.o[f / 4][4 * (f % 4) + 2], s.o[f / 4][4 * (f % 4) + 3]);
        if (lane < 32) s_ml[wave][lane] = make_float2(s.m, l);
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
        for (int i = 0; i < NF / KS; ++i) {
            const int f = stream * (NF / KS) + i;
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
        if (stream == 0) put_ml(a, v, rb, lane, m == -INFINITY ? 0.0f : m, den);
    }
}

// More than 32 rows: RB = 4 or 2 row blocks, the four waves fill each 64-key
// tile together and its 4 / RB streams take 64 / (4 / RB) of its keys.
template <int D, int RB>
__device__ __forceinline__ void run_shared(const PagedAttnArgs& a, const ItemView& v, uint16_t* s_a, uint16_t* s_b,
                                           uint32_t* s_tab, float2 (*s_ml)[32], float scale_log2, RowView rv) {
    using P = PaShape<D>;
    constexpr int KS = 4 / RB, NB = 2 / KS, LOADS = 2 * P::HALF_LOADS / 4;  // per wave, tile and tensor
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 31, kg = lane >> 5, rb = wave % RB, stream = wave / RB;
    const uint32_t per_shift = 6 - v.src.entry_shift, chunk = kTabEntries >> per_shift;

    // This lane's bytes of a load instruction's rows, blocks wave + 4j.
    const int lr = lane / P::CPR, phys = lane % P::CPR;
    const uint32_t koff = lr * v.src.row_bytes + 16 * (phys ^ pk_swz<D>(P::RI * wave + lr));
    const uint32_t voff = lr * v.src.row_bytes + 16 * (phys ^ pv_swz<D>(lr));
    static_assert((4 * P::RI) % (D / 8) == 0, "a wave's blocks share one swizzle");
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
    rv.pos = v.it.pos0 + (int32_t)((v.it.row0 + row) / v.group);
    rv.first = v.it.pos0 + (int32_t)((v.it.row0 + w_first) / v.group);
    rv.last = v.it.pos0 + (int32_t)((v.it.row0 + w_last) / v.group);
    const bool live = rb * 32 < (int)v.it.rows;
    bf16x8_t qf[P::KSTEPS];
    load_rows<D>(qf, a, v, row, kg);
    RowState<D> s;
    clear(s);

    for (uint32_t c0 = v.it.tile_begin; c0 < v.it.tile_end; c0 += chunk) {
        const uint32_t c1 = min(v.it.tile_end, c0 + chunk);
        __syncthreads();  // the last chunk's page numbers and tiles are done with
        fill_table(v, s_tab, c0, c1);
        __syncthreads();
        auto pages_of = [&](uint32_t t) __attribute__((always_inline)) {
            return s_tab[((t - c0) << per_shift) + (lane & ((1u << per_shift) - 1))];
        };
        auto fill = [&](uint32_t t, uint32_t pages, uint16_t* buf) __attribute__((always_inline)) {
            const uint32_t k0 = v.src.key0(t);
#pragma unroll
            for (int j = 0; j < LOADS; ++j) {
                const int blk = wave + 4 * j, r = P::RI * blk;
                load_lds16(row_rsrc<D>(v.src, v.src.k, pages, r >> v.src.entry_shift, k0 + r), buf + 512 * blk, koff);
                load_lds16(row_rsrc<D>(v.src, v.src.v, pages, r >> v.src.entry_shift, k0 + r), buf + 64 * D + 512 * blk,
                           voff);
            }
        };
        uint32_t pages = pages_of(c0);
        fill(c0, pages, s_a);
        pages = pages_of(min(c0 + 1, c1 - 1));
        __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
        __syncthreads();
        // Tile t from `cur` while tile t + 1 streams into `nxt`, whose last
        // readers passed the previous barrier.  The wait for the loads is
        // explicit: the compiler's tracking of loads that write LDS is not
        // relied on.
        auto step = [&](uint32_t t, const uint16_t* cur, uint16_t* nxt) __attribute__((always_inline)) {
            if (t + 1 < c1) {
                fill(t + 1, pages, nxt);
                pages = pages_of(min(t + 2, c1 - 1));
            }
            const uint32_t k0 = v.src.key0(t) + 32 * NB * stream;
            if (live && !rv.none(k0, k0 + 32 * NB - 1))
                tile<D, NB>(s, cur + 32 * NB * stream * D, cur + (64 + 32 * NB * stream) * D, k_off, v_off, qf, rv, k0,
                            v.src.key_end, scale_log2, kg);
            __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);
            __syncthreads();
        };
        for (uint32_t t = c0; t < c1; t += 2) {
            step(t, s_a, s_b);
            if (t + 1 < c1) step(t + 1, s_b, s_a);
        }
    }
    finish<D, KS>(a, v, s, s_a, s_b, s_ml, wave, lane);
}

// Up to 32 rows: wave w streams the 32-key halves w, w + 4, ... of the tiles.
template <int D>
__device__ __forceinline__ void run_streams(const PagedAttnArgs& a, const ItemView& v, uint16_t* s_a, uint16_t* s_b,
                                            uint32_t* s_tab, float2 (*s_ml)[32], float scale_log2, RowView rv) {
    using P = PaShape<D>;
    constexpr int NL = P::HALF_LOADS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 31, kg = lane >> 5;
    const uint32_t per_shift = 6 - v.src.entry_shift, chunk = kTabEntries >> per_shift;
    uint16_t* const sk = s_a + wave * 32 * D;
    uint16_t* const sv = s_b + wave * 32 * D;

    const int lr = lane / P::CPR, phys = lane % P::CPR;
    constexpr int SWZ = D / 8 / P::RI;  // instructions after which K's swizzle repeats
    uint32_t koff[SWZ];
#pragma unroll
    for (int j = 0; j < SWZ; ++j) koff[j] = lr * v.src.row_bytes + 16 * (phys ^ pk_swz<D>(P::RI * j + lr));
    const uint32_t voff = lr * v.src.row_bytes + 16 * (phys ^ pv_swz<D>(lr));
    int k_off[P::KSTEPS], v_off[P::DBLK];
#pragma unroll
    for (int ks = 0; ks < P::KSTEPS; ++ks) k_off[ks] = ql * D + 8 * ((2 * ks + kg) ^ pk_swz<D>(ql));
    {
        const int s16 = lane & 15, g16 = lane >> 4, vrow = 4 * kg + (s16 >> 2);
#pragma unroll
        for (int db = 0; db < P::DBLK; ++db)
            v_off[db] = vrow * D + 8 * ((4 * db + 2 * (g16 & 1) + ((s16 & 3) >> 1)) ^ pv_swz<D>(vrow)) + 4 * (s16 & 1);
    }
    const uint32_t last_row = v.it.rows - 1, row = min((uint32_t)ql, last_row);
    rv.pos = v.it.pos0 + (int32_t)((v.it.row0 + row) / v.group);
    rv.first = v.it.pos0 + (int32_t)(v.it.row0 / v.group);
    rv.last = v.it.pos0 + (int32_t)((v.it.row0 + last_row) / v.group);
    bf16x8_t qf[P::KSTEPS];
    load_rows<D>(qf, a, v, row, kg);
    RowState<D> s;
    clear(s);

    for (uint32_t c0 = v.it.tile_begin; c0 < v.it.tile_end; c0 += chunk) {
        const uint32_t c1 = min(v.it.tile_end, c0 + chunk);
        __syncthreads();
        fill_table(v, s_tab, c0, c1);
        __syncthreads();
        auto pages_of = [&](uint32_t h) __attribute__((always_inline)) {
            return s_tab[(((h >> 1) - c0) << per_shift) + (lane & ((1u << per_shift) - 1))];
        };
        auto key_of = [&](uint32_t h) __attribute__((always_inline)) { return v.src.key0(h >> 1) + 32 * (h & 1); };
        auto fill_k = [&](uint32_t h, uint32_t pages) __attribute__((always_inline)) {
            const uint32_t k0 = key_of(h), r0 = 32 * (h & 1);
#pragma unroll
            for (int j = 0; j < NL; ++j)
                load_lds16(row_rsrc<D>(v.src, v.src.k, pages, (r0 + P::RI * j) >> v.src.entry_shift, k0 + P::RI * j),
                           sk + 512 * j, koff[j % SWZ]);
        };
        auto fill_v = [&](uint32_t h, uint32_t pages) __attribute__((always_inline)) {
            const uint32_t k0 = key_of(h), r0 = 32 * (h & 1);
#pragma unroll
            for (int j = 0; j < NL; ++j)
                load_lds16(row_rsrc<D>(v.src, v.src.v, pages, (r0 + P::RI * j) >> v.src.entry_shift, k0 + P::RI * j),
                           sv + 512 * j, voff);
        };
        const uint32_t end = 2 * c1;
        uint32_t h = 2 * c0 + wave;
        if (h < end) {
            const uint32_t pages = pages_of(h);
            fill_k(h, pages);
            fill_v(h, pages);
        }
        for (; h < end; h += 4) {
            const uint32_t next = h + 4, k0 = key_of(h);
            const bool more = next < end;
            const uint32_t pages = more ? pages_of(next) : 0;
            // K has landed (V, requested after it, may not have): its operands
            // to registers, then the next K into its place.
            __builtin_amdgcn_s_waitcnt(wait_vmcnt(NL));
            __builtin_amdgcn_sched_barrier(0);
            uint4 ka[P::KSTEPS];
#pragma unroll
            for (int ks = 0; ks < P::KSTEPS; ++ks) ka[ks] = *reinterpret_cast<const uint4*>(sk + k_off[ks]);
            __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
            __builtin_amdgcn_sched_barrier(0);
            if (more) fill_k(next, pages);
            f32x16_t st[1];
#pragma unroll
            for (int i = 0; i < 16; ++i) st[0][i] = 0.0f;
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
            __builtin_amdgcn_sched_barrier(0);
            if (hidden && k0 < v.src.key_end && rv.some_hidden(k0, min(k1, v.src.key_end - 1)) &&
                any_nonfinite<D, 1>(sv, v_off)) {
                values_isolated<D, 1>(s, sv, v_off, pf, rv, k0, kg);
                __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
                __builtin_amdgcn_sched_barrier(0);
                if (more) fill_v(next, pages);
            } else {
                uint4 va[2][P::DBLK];
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int db = 0; db < P::DBLK; ++db) va[tt][db] = v_operand<D>(sv, v_off[db], tt);
                __builtin_amdgcn_s_waitcnt(kWaitLgkm0);
                __builtin_amdgcn_sched_barrier(0);
                if (more) fill_v(next, pages);
#pragma unroll
                for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                    for (int db = 0; db < P::DBLK; ++db)
                        s.o[db] = mfma32x32x16(as_bf16x8(va[tt][db]), pf[tt], s.o[db]);
            }
        }
    }
    __syncthreads();  // every wave is done with its tiles
    finish<D, 4>(a, v, s, s_a, s_b, s_ml, wave, lane);
}

// Whether the plan was made for these arguments; a launch with another plan
// fills o with NaN.
__device__ __forceinline__ bool plan_fits(const PagedPlanHeader& want, const void* plan) {
    const uint32_t* h = static_cast<const uint32_t*>(plan);
    return scalar_load(h) == want.batch && scalar_load(h + 1) == want.num_tokens &&
           scalar_load(h + 2) == want.page_size && scalar_load(h + 3) == want.max_blocks &&
           scalar_load(h + 4) == want.window && scalar_load(h + 5) == want.sinks && scalar_load(h + 6) == want.hq &&
           scalar_load(h + 7) == want.hkv && scalar_load(h + 8) == want.d && scalar_load(h + 9) == kPagedMagic;
}

template <int D>
__global__ __launch_bounds__(kPaThreads, 2) void paged_attn_kernel(PagedAttnArgs a, float scale_log2) {
    __shared__ __align__(1024) uint16_t s_a[PaShape<D>::BUF];
    __shared__ __align__(1024) uint16_t s_b[PaShape<D>::BUF];
    __shared__ uint32_t s_tab[kTabEntries];
    __shared__ float2 s_ml[4][32];
    const uint32_t hkv = a.head.hkv, lanes = paged_lanes(hkv);
    const uint32_t kvh = blockIdx.x % hkv, l = blockIdx.x / hkv;
    if (!plan_fits(a.head, a.plan)) {
        const uint64_t n = (uint64_t)a.head.num_tokens * a.head.hq * (D / 8);
        for (uint64_t i = (uint64_t)blockIdx.x * kPaThreads + threadIdx.x; i < n; i += (uint64_t)gridDim.x * kPaThreads)
            reinterpret_cast<uint4*>(a.o)[i] = make_uint4(0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u);
        return;
    }
    const uint32_t* plan = static_cast<const uint32_t*>(a.plan);
    const uint32_t n_items = scalar_load(plan + 11);
    const uint32_t* items = plan + sizeof(PagedPlanHeader) / 4;
    RowView rv{};
    rv.window = a.head.window && a.head.window < 0x80000000u ? a.head.window : 0x80000000u;
    rv.sinks = a.head.window ? a.head.sinks : 0;
    ItemView v;
    v.kvh = kvh;
    v.group = a.head.hq / hkv;
    v.num_pages = a.num_pages;
    v.src.page_shift = 31 - __builtin_clz(a.head.page_size);
    v.src.entry_shift = min(v.src.page_shift, 6u);
    v.src.row_bytes = hkv * D * 2;
    v.src.page_bytes = 2 * a.page_stride;
    v.src.k = reinterpret_cast<const char*>(a.k_cache + (uint64_t)kvh * D);
    v.src.v = reinterpret_cast<const char*>(a.v_cache + (uint64_t)kvh * D);
    for (uint32_t round = 0;; ++round) {
        const uint32_t idx = round * lanes + (round & 1 ? lanes - 1 - l : l);
        if (idx >= n_items) {
            // An odd round's unused places are its first lanes': nothing follows.
            break;
        }
        const uint32_t* w = items + (uint64_t)idx * (sizeof(PagedItem) / 4);
        v.it.req = scalar_load(w);
        v.it.token0 = scalar_load(w + 1);
        v.it.row0 = scalar_load(w + 2);
        v.it.rows = scalar_load(w + 3);
        v.it.pos0 = (int32_t)scalar_load(w + 4);
        v.src.key_end = scalar_load(w + 5);
        v.src.low_tile = scalar_load(w + 6);
        v.src.sink_tiles = scalar_load(w + 7);
        v.it.tile_begin = scalar_load(w + 8);
        v.it.tile_end = scalar_load(w + 9);
        v.it.partial = scalar_load(w + 10);
        v.table = a.block_tables + (uint64_t)v.it.req * a.head.max_blocks;
        if (v.it.rows > 64)
            run_shared<D, 4>(a, v, s_a, s_b, s_tab, s_ml, scale_log2, rv);
        else if (v.it.rows > 32)
            run_shared<D, 2>(a, v, s_a, s_b, s_tab, s_ml, scale_log2, rv);
        else
            run_streams<D>(a, v, s_a, s_b, s_tab, s_ml, scale_log2, rv);
        __syncthreads();
    }
}

// Merge of the pieces of each split 32-row block: a workgroup takes one d-block
// of one row block, its waves every fourth piece, and the four partial merges
// meet in LDS.
constexpr uint32_t kMergeWgs = 512;

template <int D>
__global__ __launch_bounds__(kPaThreads) void paged_merge_kernel(PagedAttnArgs a) {
    constexpr int DBLK = D / 32, NF = PaShape<D>::NF, U = 4;
    __shared__ float4 s_o[4][4][64];
    __shared__ float2 s_ml[4][64];
    if (!plan_fits(a.head, a.plan)) return;
    const uint32_t* plan = static_cast<const uint32_t*>(a.plan);
    const uint32_t hkv = a.head.hkv, group = a.head.hq / hkv, blocks = scalar_load(plan + 12);
    const PagedPlanLayout lay = paged_plan_layout(a.head.batch, a.head.num_tokens, a.head.hq, hkv);
    const PagedSplitBlock* split =
        reinterpret_cast<const PagedSplitBlock*>(static_cast<const char*>(a.plan) + lay.split_blocks);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (uint32_t i = blockIdx.x; i < blocks * hkv * DBLK; i += gridDim.x) {
        const uint32_t db = i % DBLK, kvh = i / DBLK % hkv;
        const PagedSplitBlock sb = split[i / (DBLK * hkv)];
        const uint64_t b0 = (uint64_t)kvh * paged_partial_blocks(hkv) + sb.first;
        const bool has = (uint32_t)(lane & 31) < sb.rows;
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
        if (has) {
            const uint32_t r = sb.row0 + (lane & 31), token = sb.token0 + r / group, head = kvh * group + r % group;
            const float inv = tot == 0.0f ? 0.0f : 1.0f / tot;
            uint16_t* o = a.o + ((uint64_t)token * a.head.hq + head) * D + 32 * db + 8 * wave + 4 * (lane >> 5);
            *reinterpret_cast<uint2*>(o) =
                make_uint2(pack_bf16x2(x.x * inv, x.y * inv), pack_bf16x2(x.z * inv, x.w * inv));
        }
    }
}

template <int D>
hipError_t launch_attn_t(const PagedAttnArgs& a, hipStream_t st) {
    const uint32_t wgs = a.head.hkv * paged_lanes(a.head.hkv);
    hipLaunchKernelGGL((paged_attn_kernel<D>), dim3(wgs), dim3(kPaThreads), 0, st, a, kLog2e / sqrtf((float)D));
    if (hipError_t e = hipGetLastError()) return e;
    hipLaunchKernelGGL((paged_merge_kernel<D>), dim3(kMergeWgs), dim3(kPaThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
    return a.head.d == 64 ? launch_attn_t<64>(a, stream) : launch_attn_t<128>(a, stream);
}

}  // namespace tiattn
