// Rows of the paged 8-bit cache (fp8.hpp has its format): written by the
// pre-attention pass, and read back to bf16.
//
// Write.  Q as in the bf16 prologue.  K (normalised, rotated) and V by blocks of
// 16 cache rows and head: with m the largest finite |x| that a call writes into a
// block, the least e with m <= 448 * 2^e is what the block needs.  A block whose
// first row is written begins anew with that e; else it has rows of earlier
// calls, its e only grows, and when it does those rows' codes are rounded again
// (exact, but for codes that get below the normal range).  Each new value is
// rounded once, to its code.
//
// Token rows of one block are neighbours, so a workgroup takes the runs of rows
// that begin among its 16 (up to 31 rows) for some heads of K or V, and no two
// workgroups share a block: no atomics, and the same bytes every time.  A row is
// in D / 16 lanes, a run's largest value goes over LDS, and nothing is read twice.
// The copies in and out bound it: 8192 tokens of 32 and 8 heads of 128 move 189 MB
// in 40 us, 4.7 TB/s (the bf16 prologue, 201 MB, takes 37; Q's part has the registers of
// K's, four waves a SIMD).  Few tokens wait for a chain of latencies: slots, rows, LDS,
// codes; 4 us.  Where a block grows its other rows follow, each read, rounded and
// written before the next: 9 to 13 us for 1 to 256 tokens, and of normal values a step of
// eight requests with eight heads nearly always has such a block.
//
// Read.  code * 2^e is exact in bf16.  A thread has eight values of four heads, so
// that their loads are under way together.  16 requests of up to 8192 tokens, 8 heads
// of 128: 520 MB in 95 us, 5.5 TB/s, a large copy's rate.
#include <math.h>

#include "common.hpp"
#include "fp8.hpp"
#include "paged.hpp"
#include "paged_rows.hpp"

namespace tiattn {
namespace {

constexpr int kWindow = 16;  // token rows whose runs a workgroup takes
constexpr uint32_t kWriteWgs = 512;  // two per compute unit

// The largest of a row's lanes' values, in each of them.
template <int D>
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, dpp_f32<kDppXor1>(x));
    x = fmaxf(x, dpp_f32<kDppXor2>(x));
    if constexpr (D == 128) x = fmaxf(x, dpp_f32<kDppRowHalfMirror>(x));
    return x;
}

template <uint32_t CTRL>
__device__ __forceinline__ double dpp_f64(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __float_as_uint(dpp_f32<CTRL>(__uint_as_float((uint32_t)b)));
    const uint32_t hi = __float_as_uint(dpp_f32<CTRL>(__uint_as_float((uint32_t)(b >> 32))));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// x for a later rounding to a code: 20 bits behind the point, the last one set if
// anything follows, so that halves between codes stay what they are.
__device__ __forceinline__ float sticky_f32(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x);
    const uint32_t hi = (uint32_t)(b >> 32) | ((uint32_t)b != 0 ? 1u : 0u);
    return (float)__builtin_bit_cast(double, (uint64_t)hi << 32);
}

// norm_rope_f32 in 64 bits: what it gives rounds to the code that the exact value
// rounds to, but for values within 2^-48 of a border.  (In 32 bits throughout, one of
// 2 million values got its neighbour's code.  8192 tokens of 32 and 8 heads of 128
// took 39.0 us so, and 40.1 with all but the product below in 64 bits, of 8 and 8 heads
// 24.8 and 27.0.)  The product of a value and its weight too: 32 bits hold it exactly in
// their range only, which two bf16 leave at both ends where the norm's result does not.
// (That costs 38.5 -> 39.0 us of those tokens on another card, and 28.2 -> 29.2.)
//
// The results come times 2^-kKeysDown, in fp32: a finite weight's can pass fp32's range
// and have to be the largest code then, not NaN (they are below 2^133: a row's largest
// value is at most sqrt(D) times the mean's root), and what 2^-126 cuts off at the other
// end has the code 0, whose values end at 2^-110 = 2^kFp8Low * 2^-10.
constexpr int kKeysDown = 16;
template <int D>
__device__ __forceinline__ void norm_rope_f64(uint4 xr, uint4 xi, uint4 wr, uint4 wi, const float4 (&rope)[4], float eps,
                                              float (&re)[8], float (&im)[8]) {
    // (Keeps a loop's angles and weights, and the values over the sum, from being held converted.)
    float4 cs[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        cs[k] = rope[k];
        asm volatile("" : "+v"(cs[k].x), "+v"(cs[k].y), "+v"(cs[k].z), "+v"(cs[k].w));
    }
    asm volatile("" : "+v"(wr.x), "+v"(wr.y), "+v"(wr.z), "+v"(wr.w), "+v"(wi.x), "+v"(wi.y), "+v"(wi.z), "+v"(wi.w));
    bf16x8_to_f32(xr, re);
    bf16x8_to_f32(xi, im);
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fma((double)re[k], (double)re[k], fma((double)im[k], (double)im[k], ss));
    ss += dpp_f64<kDppXor1>(ss);
    ss += dpp_f64<kDppXor2>(ss);
    if constexpr (D == 128) ss += dpp_f64<kDppRowHalfMirror>(ss);
    const double inv = rsqrt(ss * (1.0 / D) + (double)eps) * (1.0 / (1 << kKeysDown));
#pragma unroll
    for (int k = 0; k < 8; ++k) asm volatile("" : "+v"(re[k]), "+v"(im[k]));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint32_t gr = word_of(wr, k / 2), gi = word_of(wi, k / 2);
        const double r = (double)re[k] * (k % 2 ? bf16_hi(gr) : bf16_lo(gr));
        const double i = (double)im[k] * (k % 2 ? bf16_hi(gi) : bf16_lo(gi));
        const double c = k % 2 ? cs[k / 2].z : cs[k / 2].x, s = k % 2 ? cs[k / 2].w : cs[k / 2].y;
        re[k] = sticky_f32((c * r - s * i) * inv);
        im[k] = sticky_f32((c * i + s * r) * inv);
    }
}

// By one workgroup: heads [head0, head1) of K or V in a window's runs, PARTS heads
// at a time, HALVES waves each, of which one has the first 64 / (D / 16) rows of a
// group and the other the rest.  (Both in one wave: 4 us longer at 8192 tokens.)
template <int D>
struct WriteShape {
    static constexpr int LPR = D / 16, RPP = 64 / LPR, HALVES = kWindow / RPP, PARTS = 4 / HALVES;
};
struct WriteLds {
    float most[2][4][32];
    uint32_t bit[4][32];
};
template <int D>
__device__ __forceinline__ void write_blocks(const PagedPrologueFp8Args& a, uint32_t window, bool is_k, uint32_t head0,
                                             uint32_t head1, WriteLds& lds) {
    typedef WriteShape<D> W;
    constexpr int LPR = W::LPR, HALF = D / 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c = lane % LPR;
    const int local = wave / W::HALVES, g = wave % W::HALVES * W::RPP + lane / LPR;
    // Lane i + 1 looks at row i of the 32 from the window's first on, lane 0 at
    // the one before.
    const int64_t look = (int64_t)window * kWindow + lane - 1;
    const bool looks = look >= 0 && look < a.num_tokens && lane <= 32;
    const uint32_t slot_at = looks ? a.slots[look] : kNoSlot;
    const uint32_t pos_at = looks && is_k ? min(a.positions[look], a.num_positions - 1) : 0;
    const bool live = slot_at < a.num_slots;
    const uint32_t block = live ? slot_at / kFp8Block : kNoSlot, before = __shfl_up(block, 1);
    const uint32_t has = (uint32_t)(__ballot(live) >> 1);                       // rows with a slot
    const uint32_t first = (uint32_t)(__ballot(live && block != before) >> 1);  // of a run
    const uint32_t own = first & ((1u << kWindow) - 1);
    if (!own) return;
    const uint32_t edges = ~has | first, past = edges & ~((1u << kWindow) - 1);
    const int end = past ? __builtin_ctz(past) : 32;

    uint8_t* const cache = is_k ? a.k_cache : a.v_cache;
    const uint16_t* from = a.v;
    asm("" : "+s"(from));  // (or the choice is made through scratch memory)
    if (is_k) from = a.k;
    const uint32_t in_page = (1u << a.page_shift) - 1;
    const int down = is_k ? kKeysDown : 0;
    uint4 wr = make_uint4(0, 0, 0, 0), wi = wr;
    if (is_k) {
        wr = ldg16(a.k_weight + 8 * c);
        wi = ldg16(a.k_weight + 8 * c + HALF);
    }
    // Whole runs, up to 16 rows, at a time: a prompt's block, sixteen decoded tokens.
    // (The same groups in all waves, whose heads differ only.)
    for (int begin = __builtin_ctz(own), next; begin < end; begin = next) {
        const uint64_t cuts = ((uint64_t)edges | 1ull << end) & ((2ull << min(begin + kWindow, end)) - (2ull << begin));
        next = cuts ? 63 - __builtin_clzll(cuts) : min(begin + kWindow, end);
        const int i = begin + g;
        const bool mine = i < next && (has >> i & 1);
        const uint32_t slot = __shfl(slot_at, min(i, 31) + 1), pos = __shfl(pos_at, min(i, 31) + 1);
        const uint32_t row = slot & in_page, rows = in_page + 1;
        uint8_t* const page = cache + (mine ? (uint64_t)(slot >> a.page_shift) * a.page_bytes : 0);
        float* const scales = reinterpret_cast<float*>(page + (uint64_t)a.hkv * D * rows) + (mine ? row / kFp8Block : 0);
        const uint16_t* const src = from + (mine ? ((uint64_t)window * kWindow + i) * a.hkv * D + 8 * c : 0);
        float4 cs[4];
        if (is_k && mine) {
            const float4* const rope = reinterpret_cast<const float4*>(a.rope + (uint64_t)pos * D + 16 * c);
#pragma unroll
            for (int k = 0; k < 4; ++k) cs[k] = rope[k];
        }
        // The row's run.
        const int lead = mine ? max(begin, 31 - __builtin_clz(first & (~0u >> (31 - i)))) : 0;
        const uint32_t after = i >= 31 ? 0 : edges & (~0u << (i + 1));
        const int stop = min(next, after ? __builtin_ctz(after) : 32);
        uint32_t written = 0;

        uint4 xr, xi;
        float old_next;
        auto load = [&](uint32_t head) __attribute__((always_inline)) {
            const uint64_t h = min(head, a.hkv - 1);
            xr = ldg16_nt(src + h * D);
            xi = ldg16_nt(src + h * D + HALF);
            old_next = scales[h * (rows / kFp8Block)];
        };
        uint32_t head = head0 + local;
        load(head);
        for (int buf = 0; head - local < head1; head += W::PARTS, buf ^= 1) {
            float re[8], im[8];
            const float old = old_next;
            if (is_k) {
                norm_rope_f64<D>(xr, xi, wr, wi, cs, a.eps, re, im);
            } else {
                bf16x8_to_f32(xr, re);
                bf16x8_to_f32(xi, im);
            }
            if (head - local + W::PARTS < head1) load(head + W::PARTS);
            const bool active = mine && head < head1;
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float x = fabsf(re[k]), y = fabsf(im[k]);
                most = fmaxf(most, x < INFINITY ? x : 0.0f);
                most = fmaxf(most, y < INFINITY ? y : 0.0f);
            }
            most = row_max<D>(most);
            if (c == 0 && active) {
                lds.most[buf][local][i] = most;
                lds.bit[local][i] = 1u << (row % kFp8Block);
            }
            float was_scale = old;
            asm volatile("" : "+v"(was_scale));  // (has arrived before another wave writes the block's scale)
            __syncthreads();
            if (!active) continue;
            most = 0.0f;
            written = 0;
            for (int j = lead; j < stop; ++j) {
                most = fmaxf(most, lds.most[buf][local][j]);
                written |= lds.bit[local][j];
            }
            const bool opens = (written & 1) || !fp8_scale_valid(was_scale);
            const int need = fp8_exponent_for(most, down), was = (int)(__float_as_uint(was_scale) >> 23) - 127;
            const int e = opens ? need : max(need, was);
            const float inv = fp8_scale(down - e);
            uint8_t* const codes = page + (uint64_t)head * rows * D;
            uint8_t* const to = codes + row * D + 8 * c;
            *reinterpret_cast<uint2*>(to) = make_uint2(fp8x4_of(re[0], re[1], re[2], re[3], inv),
                                                       fp8x4_of(re[4], re[5], re[6], re[7], inv));
            *reinterpret_cast<uint2*>(to + HALF) = make_uint2(fp8x4_of(im[0], im[1], im[2], im[3], inv),
                                                              fp8x4_of(im[4], im[5], im[6], im[7], inv));
            if (i != lead) continue;
            if (c == 0) scales[(uint64_t)head * (rows / kFp8Block)] = fp8_scale(e);
            if (opens || e == was) continue;
            // The block's other rows under its larger scale.
            for (uint32_t r = 0; r < kFp8Block; ++r) {
                if (written >> r & 1) continue;
                uint4* const at = reinterpret_cast<uint4*>(codes + ((row & ~(kFp8Block - 1)) + r) * D + 16 * c);
                const uint4 w = *at;
                auto again = [&](uint32_t x) __attribute__((always_inline)) {
                    const uint32_t lo = fp8x2_to_bf16<false>(x, was_scale), hi = fp8x2_to_bf16<true>(x, was_scale);
                    return fp8x4_of(bf16_lo(lo), bf16_hi(lo), bf16_lo(hi), bf16_hi(hi), fp8_scale(-e));
                };
                *at = make_uint4(again(w.x), again(w.y), again(w.z), again(w.w));
            }
        }
        __syncthreads();  // (the next group's rows have other places, but its first head may be this one's buffer)
    }
}

// Workgroups [0, kv_wgs) write K and V, the others Q, a wave R times 64 / (D / 16)
// heads of a token.
template <int D, int R>
__global__ __launch_bounds__(256) void paged_prologue_fp8_kernel(PagedPrologueFp8Args a, uint32_t kv_wgs, uint32_t kv_parts,
                                                                uint32_t kv_heads, uint32_t q_parts) {
    constexpr int LPR = D / 16, G = 64 / LPR, HALF = D / 2;
    __shared__ WriteLds lds;
    if (blockIdx.x < kv_wgs) {
        const uint32_t part = blockIdx.x % (2 * kv_parts), head0 = part / 2 * kv_heads;
        write_blocks<D>(a, blockIdx.x / (2 * kv_parts), part % 2 == 0, head0, min(head0 + kv_heads, a.hkv), lds);
        return;
    }
    const uint32_t unit = (blockIdx.x - kv_wgs) * 4 + (threadIdx.x >> 6), t = unit / q_parts;
    if (t >= a.num_tokens) return;
    const int lane = threadIdx.x & 63, c = lane % LPR;
    const uint32_t head0 = unit % q_parts * (G * R) + lane / LPR;
    const uint32_t pos = min(a.positions[t], a.num_positions - 1);
    const uint64_t at0 = (uint64_t)t * a.hq * D + 8 * c;
    uint4 xr[R], xi[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint64_t at = at0 + (uint64_t)min(head0 + G * r, a.hq - 1) * D;
        xr[r] = ldg16_nt(a.q + at);
        xi[r] = ldg16_nt(a.q + at + HALF);
    }
    const uint4 wr = ldg16(a.q_weight + 8 * c), wi = ldg16(a.q_weight + 8 * c + HALF);
    const float4* const rope = reinterpret_cast<const float4*>(a.rope + (uint64_t)pos * D + 16 * c);
    float4 cs[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) cs[k] = rope[k];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float re[8], im[8];
        norm_rope_f32<D>(xr[r], xi[r], wr, wi, cs, a.eps, re, im);
        if (head0 + G * r < a.hq) {
            uint16_t* const to = a.q_out + at0 + (uint64_t)(head0 + G * r) * D;
            stg16_nt(to, pack_bf16x8(re));
            stg16_nt(to + HALF, pack_bf16x8(im));
        }
    }
}

template <int D>
hipError_t launch_prologue_t(const PagedPrologueFp8Args& a, hipStream_t st) {
    typedef WriteShape<D> W;
    const uint32_t windows = (a.num_tokens + kWindow - 1) / kWindow;
    // Heads of K or V that a workgroup takes one after the other, the next one's rows
    // on their way, as many as leave kWriteWgs workgroups.  (All heads at once, by
    // workgroups of their own: 8192 tokens of 32 and 8 heads of 128 45.4 us instead
    // of 40.5, 8 and 8 heads 32.0 instead of 27.3, 2048 tokens 14.0 instead of 12.6.
    // Few tokens have to be at once: then there are compute units for all.)
    uint32_t kv_heads = W::PARTS;
    while (kv_heads < a.hkv && (uint64_t)windows * 2 * ((a.hkv + 2 * kv_heads - 1) / (2 * kv_heads)) >= kWriteWgs) kv_heads *= 2;
    const uint32_t kv_parts = (a.hkv + kv_heads - 1) / kv_heads, kv_wgs = windows * 2 * kv_parts;
    // A token's heads of Q, 64 / (D / 16) to a wave's load: four loads under way, but
    // for so few heads that one has them all.  (One load a wave against four: 8192
    // tokens of 32 heads 44.7 and 40.5 us, of 16 33.9 and 31.2, of 8 26.3 and 27.3;
    // 1371 tokens of 16 9.4 and 9.6.  Loads past a token's heads repeat the last one's:
    // two of the four with 16 heads of 128.)
    constexpr uint32_t per_load = 64 / (D / 16);
    const bool many = a.hq > per_load;
    const uint32_t q_heads = (many ? 4 : 1) * per_load, q_parts = (a.hq + q_heads - 1) / q_heads;
    const uint32_t q_wgs = (uint32_t)(((uint64_t)a.num_tokens * q_parts + 3) / 4);
    if (many)
        hipLaunchKernelGGL((paged_prologue_fp8_kernel<D, 4>), dim3(kv_wgs + q_wgs), dim3(256), 0, st, a, kv_wgs, kv_parts,
                           kv_heads, q_parts);
    else
        hipLaunchKernelGGL((paged_prologue_fp8_kernel<D, 1>), dim3(kv_wgs + q_wgs), dim3(256), 0, st, a, kv_wgs, kv_parts,
                           kv_heads, q_parts);
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
