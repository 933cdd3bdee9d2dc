// Rows of the paged 8-bit cache (fp8.hpp has its format): written by the
// pre-attention pass, and read back to bf16.
//
// Write.  Q as in the bf16 prologue.  K (normalised, rotated) and V by blocks of
// 16 cache rows and head: with m the largest finite |x| that a call writes into a
// block, the least e with m <= 448 * 2^e is what the block needs.  A block whose
// first row is written begins anew with that e; else it has rows of earlier
// calls, its e only grows, and when it does those rows' codes are rounded again
// (exact, but for codes that get below the normal range).  Each new value is
// rounded once, from fp32 to its code.
//
// Token rows of one block are neighbours, so a wave takes the runs of rows that
// begin among its 16 (up to 31 rows), for one head of K or V, and no two waves
// share a block: no atomics, and the same bytes every time.
//
// Read.  code * 2^e is exact in bf16.
#include <math.h>

#include "common.hpp"
#include "fp8.hpp"
#include "paged.hpp"
#include "paged_rows.hpp"

namespace tiattn {
namespace {

constexpr int kWindow = 16;  // token rows whose runs a wave takes

// The largest of a row's lanes' values, in each of them.
template <int D>
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, dpp_f32<kDppXor1>(x));
    x = fmaxf(x, dpp_f32<kDppXor2>(x));
    if constexpr (D == 128) x = fmaxf(x, dpp_f32<kDppRowHalfMirror>(x));
    return x;
}

template <int D>
__device__ __forceinline__ void write_blocks(const PagedPrologueFp8Args& a, uint32_t window, uint32_t part,
                                             float* s_most, uint32_t* s_bit) {
    constexpr int LPR = D / 16, RPP = 64 / LPR, PASSES = 32 / RPP, HALF = D / 2;
    const int lane = threadIdx.x & 63, g = lane / LPR, c = lane % LPR;
    const bool is_k = part < a.hkv;
    const uint32_t head = is_k ? part : part - a.hkv;
    // Lane i + 1 looks at row i of the 32 from the window's first on, lane 0 at
    // the one before.
    const int64_t look = (int64_t)window * kWindow + lane - 1;
    const uint32_t slot_at = look >= 0 && look < a.num_tokens && lane <= 32 ? a.slots[look] : kNoSlot;
    const bool live = slot_at < a.num_slots;
    const uint32_t block = live ? slot_at / kFp8Block : kNoSlot, before = __shfl_up(block, 1);
    const uint32_t has = (uint32_t)(__ballot(live) >> 1);                         // rows with a slot
    const uint32_t first = (uint32_t)(__ballot(live && block != before) >> 1);    // of a run
    const uint32_t own = first & ((1u << kWindow) - 1);
    if (!own) return;
    const uint32_t past = (~has | first) & ~((1u << kWindow) - 1);
    const int begin = __builtin_ctz(own), end = past ? __builtin_ctz(past) : 32;

    const uint16_t* const src = is_k ? a.k : a.v;
    const uint16_t* const weight = is_k ? a.k_weight : nullptr;
    uint8_t* const cache = is_k ? a.k_cache : a.v_cache;
    uint4 wr = make_uint4(0, 0, 0, 0), wi = wr;
    if (is_k) {
        wr = ldg16(weight + 8 * c);
        wi = ldg16(weight + 8 * c + HALF);
    }
    float re[PASSES][8], im[PASSES][8], old[PASSES];
    uint32_t slot[PASSES];
    bool mine[PASSES];
    uint4 xr[PASSES], xi[PASSES];
    const uint32_t in_page = (1u << a.page_shift) - 1;
    auto page_at = [&](uint32_t s) __attribute__((always_inline)) {
        return cache + (uint64_t)(s >> a.page_shift) * a.page_bytes;
    };
    auto scale_at = [&](uint32_t s) __attribute__((always_inline)) {
        const uint64_t codes = (uint64_t)a.hkv * D << a.page_shift;
        return reinterpret_cast<float*>(page_at(s) + codes) + (uint64_t)head * ((in_page + 1) / kFp8Block) +
               (s & in_page) / kFp8Block;
    };
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        const int i = begin + RPP * p + g;
        mine[p] = i < end && (has >> i & 1);
        slot[p] = __shfl(slot_at, min(i, 31) + 1);
        if (!mine[p]) continue;
        const uint64_t row = (uint64_t)window * kWindow + i;
        const uint16_t* const from = src + (row * a.hkv + head) * D;
        xr[p] = ldg16_nt(from + 8 * c);
        xi[p] = ldg16_nt(from + 8 * c + HALF);
        old[p] = *scale_at(slot[p]);
    }
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        if (!mine[p]) continue;
        const int i = begin + RPP * p + g;
        if (is_k) {
            const uint32_t pos = min(a.positions[(uint64_t)window * kWindow + i], a.num_positions - 1);
            const float4* const rope = reinterpret_cast<const float4*>(a.rope + (uint64_t)pos * D + 16 * c);
            float4 cs[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) cs[k] = rope[k];
            norm_rope_f32<D>(xr[p], xi[p], wr, wi, cs, a.eps, re[p], im[p]);
        } else {
            bf16x8_to_f32(xr[p], re[p]);
            bf16x8_to_f32(xi[p], im[p]);
        }
        float most = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float x = fabsf(re[p][k]), y = fabsf(im[p][k]);
            most = fmaxf(most, x < INFINITY ? x : 0.0f);
            most = fmaxf(most, y < INFINITY ? y : 0.0f);
        }
        most = row_max<D>(most);
        if (c == 0) {
            s_most[i] = most;
            s_bit[i] = 1u << (slot[p] % kFp8Block);
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
        if (!mine[p]) continue;
        const int i = begin + RPP * p + g;
        // The row's run.
        const int lead = 31 - __builtin_clz(first & (~0u >> (31 - i)));
        const uint32_t after = i == 31 ? 0 : (~has | first) & (~0u << (i + 1));
        const int stop = after ? __builtin_ctz(after) : 32;
        float most = 0.0f;
        uint32_t written = 0;
        for (int j = lead; j < stop; ++j) {
            most = fmaxf(most, s_most[j]);
            written |= s_bit[j];
        }
        const bool opens = (written & 1) || !fp8_scale_valid(old[p]);
        const int need = fp8_exponent_for(most), was = (int)(__float_as_uint(old[p]) >> 23) - 127;
        const int e = opens ? need : max(need, was);
        const float inv = fp8_scale(-e);
        uint8_t* const block_rows = page_at(slot[p]) + ((((uint64_t)head << a.page_shift) + (slot[p] & in_page)) & ~(uint64_t)(kFp8Block - 1)) * D;
        uint8_t* const to = block_rows + slot[p] % kFp8Block * D + 8 * c;
        *reinterpret_cast<uint2*>(to) = make_uint2(fp8x4_of(re[p][0], re[p][1], re[p][2], re[p][3], inv),
                                                   fp8x4_of(re[p][4], re[p][5], re[p][6], re[p][7], inv));
        *reinterpret_cast<uint2*>(to + HALF) = make_uint2(fp8x4_of(im[p][0], im[p][1], im[p][2], im[p][3], inv),
                                                          fp8x4_of(im[p][4], im[p][5], im[p][6], im[p][7], inv));
        if (i != lead) continue;
        if (c == 0) *scale_at(slot[p]) = fp8_scale(e);
        if (opens || e == was) continue;
        // The block's other rows under its larger scale.
        for (uint32_t r = 0; r < kFp8Block; ++r) {
            if (written >> r & 1) continue;
            uint4* const at = reinterpret_cast<uint4*>(block_rows + r * D + 16 * c);
            uint4 w = *at;
            auto again = [&](uint32_t x) __attribute__((always_inline)) {
                const uint32_t lo = fp8x2_to_bf16<false>(x, old[p]), hi = fp8x2_to_bf16<true>(x, old[p]);
                return fp8x4_of(bf16_lo(lo), bf16_hi(lo), bf16_lo(hi), bf16_hi(hi), inv);
            };
            *at = make_uint4(again(w.x), again(w.y), again(w.z), again(w.w));
        }
    }
}

template <int D>
__global__ __launch_bounds__(256) void paged_prologue_fp8_kernel(PagedPrologueFp8Args a, uint32_t kv_wgs, uint32_t q_parts) {
    constexpr int LPR = D / 16, G = 64 / LPR, HALF = D / 2;
    __shared__ float s_most[4][32];
    __shared__ uint32_t s_bit[4][32];
    const int wave = threadIdx.x >> 6;
    if (blockIdx.x < kv_wgs) {
        const uint32_t unit = blockIdx.x * 4 + wave, window = unit / (2 * a.hkv);
        if (window * (uint64_t)kWindow < a.num_tokens)
            write_blocks<D>(a, window, unit % (2 * a.hkv), s_most[wave], s_bit[wave]);
        return;
    }
    const uint32_t unit = (blockIdx.x - kv_wgs) * 4 + wave, t = unit / q_parts;
    if (t >= a.num_tokens) return;
    const int lane = threadIdx.x & 63, c = lane % LPR;
    const uint32_t row = unit % q_parts * G + lane / LPR, head = min(row, a.hq - 1);
    const uint32_t pos = min(a.positions[t], a.num_positions - 1);
    const uint64_t at = ((uint64_t)t * a.hq + head) * D + 8 * c;
    const uint4 xr = ldg16_nt(a.q + at), xi = ldg16_nt(a.q + at + HALF);
    const uint4 wr = ldg16(a.q_weight + 8 * c), wi = ldg16(a.q_weight + 8 * c + HALF);
    const float4* const rope = reinterpret_cast<const float4*>(a.rope + (uint64_t)pos * D + 16 * c);
    float4 cs[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) cs[k] = rope[k];
    float re[8], im[8];
    norm_rope_f32<D>(xr, xi, wr, wi, cs, a.eps, re, im);
    if (row < a.hq) {
        stg16_nt(a.q_out + at, pack_bf16x8(re));
        stg16_nt(a.q_out + at + HALF, pack_bf16x8(im));
    }
}

template <int D>
hipError_t launch_prologue_t(const PagedPrologueFp8Args& a, hipStream_t st) {
    constexpr uint32_t G = 64 / (D / 16);
    const uint32_t q_parts = (a.hq + G - 1) / G;
    const uint64_t kv = ((uint64_t)a.num_tokens + kWindow - 1) / kWindow * 2 * a.hkv, q = (uint64_t)a.num_tokens * q_parts;
    const uint32_t kv_wgs = (uint32_t)((kv + 3) / 4);
    hipLaunchKernelGGL((paged_prologue_fp8_kernel<D>), dim3(kv_wgs + (uint32_t)((q + 3) / 4)), dim3(256), 0, st, a, kv_wgs,
                       q_parts);
    return hipGetLastError();
}

// A workgroup takes 2048 / D token rows of up to kReadHeads heads, a thread eight
// values of a row.
constexpr uint32_t kReadHeads = 4;

template <int D>
__global__ __launch_bounds__(256) void paged_read_fp8_kernel(PagedReadFp8Args a) {
    constexpr uint32_t CPR = D / 8, ROWS = 256 / CPR;
    const uint32_t t = blockIdx.x * ROWS + threadIdx.x / CPR, c = threadIdx.x % CPR;
    if (t >= min(a.num_tokens, a.query_start[a.batch])) return;
    uint32_t lo = 0, hi = a.batch;  // query_start[lo] <= t < query_start[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (a.query_start[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    const uint64_t room = (uint64_t)a.max_blocks << a.page_shift;
    const int64_t len = (int64_t)min((uint64_t)a.seq_lens[lo], room);
    const int64_t pos = len - (int64_t)a.query_start[lo + 1] + (int64_t)t;
    const bool there = pos >= 0 && pos < len;
    const uint32_t in_page = (1u << a.page_shift) - 1, row = there ? (uint32_t)pos & in_page : 0;
    const uint32_t page = there ? min(a.block_tables[(uint64_t)lo * a.max_blocks + ((uint32_t)pos >> a.page_shift)], a.num_pages - 1) : 0;
    const uint64_t base = page * a.page_bytes, scales = base + ((uint64_t)a.hkv * D << a.page_shift);
    uint2 k[kReadHeads], v[kReadHeads];
    float ks[kReadHeads], vs[kReadHeads];
    const uint32_t h0 = blockIdx.y * kReadHeads;
#pragma unroll
    for (uint32_t i = 0; i < kReadHeads; ++i) {
        const uint32_t h = min(h0 + i, a.hkv - 1);
        const uint64_t at = base + (((uint64_t)h << a.page_shift) + row) * D + 8 * c;
        const uint64_t scale = scales + ((uint64_t)h * ((in_page + 1) / kFp8Block) + row / kFp8Block) * sizeof(float);
        k[i] = *reinterpret_cast<const uint2*>(a.k_cache + at);
        v[i] = *reinterpret_cast<const uint2*>(a.v_cache + at);
        ks[i] = *reinterpret_cast<const float*>(a.k_cache + scale);
        vs[i] = *reinterpret_cast<const float*>(a.v_cache + scale);
    }
#pragma unroll
    for (uint32_t i = 0; i < kReadHeads; ++i) {
        if (h0 + i >= a.hkv) break;
        const uint64_t at = ((uint64_t)t * a.hkv + h0 + i) * D + 8 * c;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        stg16_nt(a.k_out + at, there ? fp8x8_to_bf16(k[i], ks[i]) : zero);
        stg16_nt(a.v_out + at, there ? fp8x8_to_bf16(v[i], vs[i]) : zero);
    }
}

template <int D>
hipError_t launch_read_t(const PagedReadFp8Args& a, hipStream_t st) {
    constexpr uint32_t ROWS = 2048 / D;
    const dim3 grid((a.num_tokens + ROWS - 1) / ROWS, (a.hkv + kReadHeads - 1) / kReadHeads);
    hipLaunchKernelGGL((paged_read_fp8_kernel<D>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_prologue_fp8(const PagedPrologueFp8Args& a, uint32_t d, hipStream_t stream) {
    return d == 64 ? launch_prologue_t<64>(a, stream) : launch_prologue_t<128>(a, stream);
}

hipError_t launch_paged_read_fp8(const PagedReadFp8Args& a, uint32_t d, hipStream_t stream) {
    return d == 64 ? launch_read_t<64>(a, stream) : launch_read_t<128>(a, stream);
}

}  // namespace tiattn
