// Shared by the kernels of attention of new tokens over the paged cache (chunk.hip: few rows, chunk_tiles.hip: many).
#pragma once
#include "qr_paged.h"

// n / d for n below 2^30: umulhi(4 n, inverse) >> shift
struct Divisor {
    u32 inverse, shift;
};
__device__ __forceinline__ int divided(int n, Divisor d) { return (int)(__umulhi((u32)n << 2, d.inverse) >> d.shift); }
static inline Divisor divisor_of(int64_t d) {
    const u32 log2 = d > 1 ? 64u - (u32)__builtin_clzll((unsigned long long)d - 1) : 0u;       // the least s for which 2^s reaches d
    return Divisor{(u32)(((1ull << (30 + log2)) + (uint64_t)d - 1) / (uint64_t)d), log2};
}

// What a launch works on.  Rows of a (sequence, key head): row r is new token r / group, query head kv_head * group + r % group.
struct Chunk {
    PagedKV c;
    const f16* q;
    f16* o;
    const int32_t* starts;            // nullptr: one new token per sequence
    float* part;                      // splits > 1: 132 floats per row and split: maximum, sum, -, -, 128 outputs
    int64_t q_stride, o_stride;       // halves from a token to the next
    int tokens, group, tiles, splits, window, sinks;      // window 0: none
    int q_had;
    Divisor per_group, per_split, per_head;     // of `group`, `splits`, the key heads
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kScale = 0.08838834764831845f;             // 1 / sqrt(128)
constexpr float kEmpty = -1e30f;                           // the running maximum of a row that has seen nothing
constexpr float kGrow = 8.f;                               // a maximum is raised when a logit (base 2) is this far above it

template <int MASK>
__device__ __forceinline__ u32x2 both_halves(u32 w) {      // the words of this lane and of lane ^ MASK, the lower lane's first
    if constexpr (MASK == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(w, w, false, false);
        return u32x2{(u32)r[0], (u32)r[1]};
    } else {
        const auto r = __builtin_amdgcn_permlane16_swap(w, w, false, false);
        return u32x2{(u32)r[0], (u32)r[1]};
    }
}
__device__ __forceinline__ float as_f32(u32 w) { return __builtin_bit_cast(float, w); }
__device__ __forceinline__ u32 as_u32(float v) { return __builtin_bit_cast(u32, v); }
// over the four lanes that hold a query row's quarters
__device__ __forceinline__ float quarters_sum(float v) {
    const u32x2 a = both_halves<16>(as_u32(v));
    v = as_f32(a.x) + as_f32(a.y);
    const u32x2 b = both_halves<32>(as_u32(v));
    return as_f32(b.x) + as_f32(b.y);
}
__device__ __forceinline__ float quarters_max(float v) {
    const u32x2 a = both_halves<16>(as_u32(v));
    v = __builtin_fmaxf(as_f32(a.x), as_f32(a.y));
    const u32x2 b = both_halves<32>(as_u32(v));
    return __builtin_fmaxf(as_f32(b.x), as_f32(b.y));
}

// ---- int4 operands
// The codes of a word as fp16 operands: pairs (0, 4), (1, 5), (2, 6), (3, 7).  A code in the lowest (next) four bits of a half is the subnormal number
// code 2^-24 (code 2^-20), which the matrix instructions take exactly: no conversion.  The query's dimensions come in that order, those that meet an
// upper nibble a sixteenth (exact from 2^-10 on, below in units of 2^-20), and logits take 2^24.
constexpr float kCodeUnit = 16777216.f;
constexpr u32 kNoParameters = 0x00003C00u;                 // scale 1, zero 0
__device__ __forceinline__ u32x4 codes_of(u32 w) {
    const u32 w8 = w >> 8;
    return u32x4{w & 0x000F000Fu, w & 0x00F000F0u, w8 & 0x000F000Fu, w8 & 0x00F000F0u};
}
__device__ __forceinline__ u32x4 query_for_codes(u32x4 w) {
    const f16x2 part = {(f16)0.0625f, (f16)0.0625f};
    return u32x4{__builtin_amdgcn_perm(w[2], w[0], 0x05040100u), __builtin_bit_cast(u32, as_f16x2(__builtin_amdgcn_perm(w[2], w[0], 0x07060302u)) * part),
                 __builtin_amdgcn_perm(w[3], w[1], 0x05040100u), __builtin_bit_cast(u32, as_f16x2(__builtin_amdgcn_perm(w[3], w[1], 0x07060302u)) * part)};
}
// scale = f 2^e with 1 <= |f| < 2 (e at most 12: |f| < 16 then): 2^e, 0 for a scale of zero, whose f is 1
__device__ __forceinline__ float power_of(float scale) {
    const u32 bits = as_u32(scale) & 0x7F800000u;
    return as_f32(bits > 0x45800000u ? 0x45800000u : bits);
}
__device__ __forceinline__ float factor_of(float scale, float power) { return power == 0.f ? 1.f : scale * as_f32(0x7F000000u - as_u32(power)); }
// 2^e of the scales of two {scale, zero} words, as a pair: a normal fp16 number's exponent alone.  `plain` stays set where scaled_codes takes them
// (2^-14 .. 2^5: scales below 64)
__device__ __forceinline__ u32 powers_of(u32 w0, u32 w1, bool& plain) {
    const u32 p = __builtin_amdgcn_perm(w1, w0, 0x05040100u) & 0x7C007C00u;
    plain = plain && (p & 0xFFFFu) - 0x0400u <= 0x4C00u && (p >> 16) - 0x0400u <= 0x4C00u;
    return p;
}
// weight times factor -> fp16, rounded once: two weights, two factors (a pair of fp16 numbers)
__device__ __forceinline__ u32 scaled_pair(float w0, float w1, u32 factors) {
    u32 r;
    asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "=v"(r) : "v"(w0), "v"(factors));
    asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "+v"(r) : "v"(w1), "v"(factors));
    return r;
}
// w: four codes of one vector in the low half, of another in the high half -> code 2^e of both, code by code: (1024 + code) 2^e - 1024 2^e is exact
struct CodeMasks {                     // in registers: a literal for the mask and one for the exponent are more than one instruction takes
    u32 low, high;
};
__device__ __forceinline__ CodeMasks code_masks() {
    CodeMasks m{0x000F000Fu, 0x00F000F0u};
    asm("" : "+v"(m.low), "+v"(m.high));
    return m;
}
__device__ __forceinline__ u32 and_or(u32 w, u32 mask, u32 bits) {
    u32 r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "v"(mask), "s"(bits));
    return r;
}
__device__ __forceinline__ u32x4 scaled_codes(u32 w, u32 power, CodeMasks m) {
    const u32 w8 = w >> 8;
    const f16x2 p = as_f16x2(power), lo = p * f16x2{(f16)-1024.f, (f16)-1024.f}, hi = p * f16x2{(f16)-64.f, (f16)-64.f};
    return u32x4{__builtin_bit_cast(u32, __builtin_elementwise_fma(as_f16x2(and_or(w, m.low, 0x64006400u)), p, lo)),
                 __builtin_bit_cast(u32, __builtin_elementwise_fma(as_f16x2(and_or(w, m.high, 0x54005400u)), p, hi)),
                 __builtin_bit_cast(u32, __builtin_elementwise_fma(as_f16x2(and_or(w8, m.low, 0x64006400u)), p, lo)),
                 __builtin_bit_cast(u32, __builtin_elementwise_fma(as_f16x2(and_or(w8, m.high, 0x54005400u)), p, hi))};
}
__device__ __forceinline__ u32x4 scaled_codes(u32 w, u32 power) {              // (two registers less)
    const u32 w8 = w >> 8;
    const f16x2 p = as_f16x2(power), lo = p * f16x2{(f16)-1024.f, (f16)-1024.f}, hi = p * f16x2{(f16)-64.f, (f16)-64.f};
    return u32x4{__builtin_bit_cast(u32, __builtin_elementwise_fma(as_f16x2((w & 0x000F000Fu) | 0x64006400u), p, lo)),
                 __builtin_bit_cast(u32, __builtin_elementwise_fma(as_f16x2((w & 0x00F000F0u) | 0x54005400u), p, hi)),
                 __builtin_bit_cast(u32, __builtin_elementwise_fma(as_f16x2((w8 & 0x000F000Fu) | 0x64006400u), p, lo)),
                 __builtin_bit_cast(u32, __builtin_elementwise_fma(as_f16x2((w8 & 0x00F000F0u) | 0x54005400u), p, hi))};
}
// the same for any scales (as {scale, zero} words)
__device__ __forceinline__ u32x4 scaled_codes_slow(u32 w, u32 w0, u32 w1) {
    const f16x2 p = {(f16)power_of((float)as_f16x2(w0)[0]), (f16)power_of((float)as_f16x2(w1)[0])};
    u32x4 out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2 code = {(f16)(float)(w >> (4 * i) & 15u), (f16)(float)(w >> (16 + 4 * i) & 15u)};
        out[i] = __builtin_bit_cast(u32, code * p);
    }
    return out;
}

// the new tokens of sequence b: the first one's row in q and o, how many rows there are of them (kept inside q and o, whatever the bounds say), and how many
// tokens from that row on the bounds say: those that q has no rows for are the sequence's last ones
struct Fresh {
    int start, count, all;
};
__device__ __forceinline__ Fresh fresh_of(const Chunk& a, int b) {
    if (!a.starts) return Fresh{b, 1, 1};
    int start = a.starts[b];
    const int end = a.starts[b + 1];
    start = start < 0 ? 0 : start;
    const int stop = end > a.tokens ? a.tokens : end;
    return Fresh{start, stop > start ? stop - start : 0, end > start ? end - start : 0};
}

__device__ __forceinline__ int lanes_sum(int v) {          // over the wave
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);       // row_shr 1, 2, 4, 8: a row's last lane has its sum
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);       // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return __builtin_amdgcn_readlane(v, 63);
}
// Work item `number` of a head: a sequence and one of its tiles of PER rows, last tiles (most positions) first; false: there is none.  Items without rows come
// last: between others they leave whole shader engines idle, since workgroups are handed out to them in turn (8 sequences of 2048, 1792 .. 256 tokens, 64 on 8
// heads: 528 us with them, 369 without).  Of more than 64 sequences the tiles are not counted.
template <int PER>
__device__ __forceinline__ bool item_of(const Chunk& a, int number, int& b, int& tile) {
    const int batch = a.c.batch_size;
    if (a.tiles == 1 || batch > 64) {
        tile = a.tiles == 1 ? 0 : a.tiles - 1 - number / batch;
        b = a.tiles == 1 ? number : number % batch;
        return tile * PER < fresh_of(a, b).count * a.group;
    }
    const int lane = threadIdx.x & 63;
    const int held = (fresh_of(a, lane < batch ? lane : 0).count * a.group + PER - 1) / PER;
    const int mine = lane >= batch ? 0 : held < a.tiles ? held : a.tiles;
    auto above = [&](int t) { return lanes_sum(mine > t ? mine - t : 0); };      // tiles t and higher of all sequences
    if (above(0) <= number) return false;
    int low = 0, high = a.tiles;                           // above(low) > number >= above(high)
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (above(mid) > number) low = mid;
        else high = mid;
    }
    tile = low;
    const int rank = number - above(low + 1);
    const uint64_t who = __builtin_amdgcn_ballot_w64(mine > low);
    const int before = __builtin_amdgcn_mbcnt_hi((u32)(who >> 32), __builtin_amdgcn_mbcnt_lo((u32)who, 0));
    b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(mine > low && before == rank));
    return true;
}

// The positions that the rows of a tile see, in steps of 1 << LOG: steps [0, near) hold the sinks, then [far, far + rest).
struct Steps {
    int near, far, all;
    __device__ int at(int s) const { return s < near ? s : s - near + far; }
};
template <int LOG>
__device__ __forceinline__ Steps steps_of(const Chunk& a, int lowest, int highest) {        // positions of the tile's first and last row
    Steps s{0, 0, 0};
    if (highest < 0) return s;
    int from = 0;
    if (a.window > 0 && lowest - a.window + 1 > 0) {
        from = lowest - a.window + 1;
        const int sinks = a.sinks < from ? a.sinks : from;
        s.near = (sinks + (1 << LOG) - 1) >> LOG;
    }
    s.far = from >> LOG;
    if (s.far < s.near) s.far = s.near;
    const int end = (highest >> LOG) + 1;
    s.all = s.near + (end > s.far ? end - s.far : 0);
    return s;
}

// chunk_tiles.hip
int qr_internal_chunk_tiles(bool fp16, const Chunk& a, Divisor pages, int64_t groups, hipStream_t st);
