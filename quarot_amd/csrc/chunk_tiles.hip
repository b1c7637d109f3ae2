// Attention of new tokens over the paged cache for many rows of a (sequence, key head): the mathematics of chunk.hip on tiles of 256 rows.
//
// Four waves, one per SIMD, of 64 rows each share the cached vectors of a step of 64 positions: each is unpacked once per workgroup, from
// registers into LDS, as the fp16 operand that the matrix instructions take, and each operand read from LDS serves two of them (with 32 rows
// per wave LDS was busy for longer than the matrix unit).  A wave holds the positions in its registers and the rows in its lanes (chunk.hip:
// no exchange between lanes from the first product to the second).
//
// What is not a code's is in the products too.  Of a logit: zero_j sum(q), the row's running maximum, and the logarithm of the value's factor
// f_j, so that exp2 gives weight_j f_j, which is rounded to fp16: a product of bf16 pieces that hold 24 bits together.  Of the sums: besides the
// 128 dimensions the second product's operand has the reciprocal 1 / f_j and the zero point zero_j / f_j of every position as pairs of fp16
// numbers (22 bits of each; the second ones times 2^11, so that small ones have them too), so that the sums of weights and of weights times
// zero points are those of the weights as they were rounded.  (A lane's vector unit would take as long for all this as for the exponentials.)
//
// A wave has its SIMD to itself, so the vector work is laid between the matrix instructions by hand, in slots: while the first product of the
// next 32 positions runs, the weights of these 32; while their second product runs, the logits of the next, and the unpacking of what the
// workgroup needs a step later.  2048 tokens after 30720, 64 on 8 heads: 2.31 to 2.50 ms on different cards, 850 to 920 TFLOP/s, 1000 to 1090 with the products for
// the sums and the lines; a step takes some 5000 cycles, 2432 of them matrix instructions, at the 2.0 - 2.2 GHz that its power allows (a large library product: 1140).
#include "qr_chunk.h"

namespace {

constexpr int kRows = 256, kStep = 64;
// LDS: three steps' keys (the next step's are read while others still read this one's), two steps' values
// A key's row is padded by 16 bytes, a dimension's too, and 16 more behind every 32nd, so that the reads (16 lanes of 16 bytes, rows that follow one another) and the
// writes (32 lanes of 8 bytes, rows 4, 8, 32 and 64 apart) spread over the banks, and every piece's place is one address per lane and a constant.  Of 2048 tokens after
// 30720 conflicts are 18 % of the cycles that LDS works (SQ_LDS_BANK_CONFLICT 6.5e7 of SQ_LDS_IDX_ACTIVE 3.5e8).
constexpr int kKeyRow = 272, kDimRow = 144;
__host__ __device__ constexpr int dim_row(int r) { return r * kDimRow + (r >> 5) * 16; }
constexpr int kSlope = 64 * kKeyRow, kLine = kSlope + 256, kThere = kLine + 2048, kKeys = (kThere + 8 + 511) / 512 * 512;
constexpr int kOdd = dim_row(133), kValues = (kOdd + 8 + 511) / 512 * 512;
// A row's largest weight times its value's factor lies between 2^kBase and 2^kHigh, an fp16 number: a first maximum is put at kBase, and so is one that a logit
// (base 2, with the factor) exceeds kHigh by.  Factors are below two (up to 16 only for scales from 2^13 on), so the largest weight is one at least, and the
// smallest ones are rounded in steps of 2^-24 of it; with maxima put at zero it could be a half, and the steps as much more of it (scales of 2^-24 .. 2^10, logits of
// hundreds: errors of 1.56 times what rounded weights explain).  Higher maxima leave less room until they are raised: kBase 4 and kHigh 15 took 428 us for 8 x up
// to 2048 tokens on 64 and 8 heads, these 361, 0 and 15 363.
constexpr float kHigh = 15.9f, kBase = 1.f;
constexpr int kLds = 3 * kKeys + 2 * kValues;

// What a thread has fetched for a step: four of the sixteen pieces of a key and its parameters; four positions' values in eight dimensions, their
// parameters and those of the position that has the key's number.  mask: which of the wave's sixteen positions are there.
template <bool F16>
struct KeyCodes {
    u32x4 k[F16 ? 4 : 1];
    u32 p, pv, mask;                   // pv: the value's parameters
};
template <bool F16>
struct ValueCodes {
    u32x4 v4[F16 ? 4 : 1];
    u32 v[F16 ? 1 : 4], scales[F16 ? 1 : 4], p, mask;
};

// Matrix instructions, spelled out: the first product's results and the logits' line are for the vector unit and have to lie where it reaches them, the
// second product's accumulators in the half of the register file that only matrix instructions use.  (Left to itself the compiler puts all of
// them into that half, and copies 64 values a unit back.)  It then inserts no wait states either.  A result is read by the vector unit two
// matrix instructions after its last one at the earliest (32 cycles each; it is there after 11 of 4), or behind `settled`.
__device__ __forceinline__ void mfma_first(f32x16& c, u32x4 a, u32x4 b) { asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "a"(b)); }
__device__ __forceinline__ void mfma_more(f32x16& c, u32x4 a, u32x4 b) { asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "a"(b)); }
__device__ __forceinline__ void mfma_line(f32x16& c, u32x4 a, u32x4 b) { asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(c) : "v"(a), "v"(b)); }
__device__ __forceinline__ void mfma_second(f32x16& c, u32x4 a, u32x4 b) { asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b)); }
__device__ __forceinline__ void mfma_overflow(f32x16& c, u32x4 a, u32x4 b) { asm volatile("s_nop 3\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b)); }
// a register of that half times v: where it lies (the compiler would move whole accumulators to the vector unit's half and back in every turn)
__device__ __forceinline__ void scale_accumulator(float& c, float v) {
    float t;
    asm volatile("v_accvgpr_read_b32 %1, %0\n\tv_mul_f32 %1, %1, %2\n\tv_accvgpr_write_b32 %0, %1" : "+a"(c), "=&v"(t) : "v"(v));
}
__device__ __forceinline__ void settled() { asm volatile("s_nop 15\n\ts_nop 15" ::: "memory"); }
__device__ __forceinline__ f32x16 zeros() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}
// the upper 16 bits of two floats: lo in the low half
__device__ __forceinline__ u32 tops(float lo, float hi) { return __builtin_amdgcn_perm(as_u32(hi), as_u32(lo), 0x07060302u); }
__device__ __forceinline__ float top(float v) { return as_f32(as_u32(v) & 0xFFFF0000u); }
__device__ __forceinline__ bool strange(u32 w) { return (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u; }      // a half of it is not finite

#define SLOT __builtin_amdgcn_sched_barrier(0)
#define INLINE __attribute__((always_inline))        // (what a function that is not inlined captures lies in memory)

// ALIGNED: pages of a multiple of 16 positions, so that the sixteen positions that a wave fetches lie in one page
// DEALT: one prefix's tiles, whose steps the workgroups share evenly
template <bool F16, bool ALIGNED, bool DEALT>
__device__ __forceinline__ void attend_tiles(const Chunk& a, const Divisor& pages) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const PagedKV& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int id = divided(blockIdx.x, a.per_split), item = divided(id, a.per_head);
    int split = blockIdx.x - id * a.splits, head = id - item * c.num_heads;    // neighbours are on different XCDs, a head's tiles on one where 8 divides the heads
    int b = 0, tile = 0;
    if (!DEALT && !item_of<kRows>(a, item, b, tile)) return;
    const Fresh tokens = fresh_of(a, b);
    const int rows = tokens.count * a.group;
    const int p0 = c.indptr[b], npages = c.indptr[b + 1] - p0;
    const int len = npages > 0 ? (npages - 1) * c.page_size + c.last_page_offset[b] : 0;
    const int first_place = len - tokens.all;              // the first new token's position
    const int64_t page_slots = (int64_t)c.num_layers * 2 * c.num_heads * c.page_size;
    int64_t head_slots = ((int64_t)c.layer_idx * 2 * c.num_heads + head) * c.page_size;
    const int64_t kv_slots = (int64_t)c.num_heads * c.page_size;
    constexpr uint32_t VEC = F16 ? 256 : 64;               // bytes of a vector

    // Dealt out: the steps of all heads' tiles, one behind the other, in equal shares (544 tiles on 256 CUs: 2.1 turns of a tile's steps, where whole tiles take 3 and
    // fourths of them 2.25 and twice the states).  An XCD has shares that follow one another, of few heads.  A tile's shares are its states 0, 1, ..., and
    // whoever has its last step marks those that there are not as empty.
    int done = 0;                                          // of the workgroup's share

    // what never changes: the values' operand beyond row 131 (fp16 pages: beyond 127, with a row of ones for the weights' sum), the second half of the logits'
    // line, whose first factor is one
    if (tid < 2 * 40) {
        const int at = tid % 40;
        *(u32x4*)(lds + 3 * kKeys + (tid < 40 ? 0 : kValues) + dim_row(128) + (at >> 3) * kDimRow + (at & 7) * 16) = F16 && at < 8 ? u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u} : u32x4{0, 0, 0, 0};
    }
    if (tid < 3 * 64) *(u32x4*)(lds + (tid >> 6) * kKeys + kLine + 1024 + (tid & 63) * 16) = u32x4{0x00003F80u, 0, 0, 0};

    // ---- a step's way into LDS.  Thread (key, e) takes pieces e, e + 4, e + 8, e + 12 of a key (int4: the words 4 e .. 4 e + 3); thread (four positions,
    // word) their values in dimensions 8 word ...  The four positions are 16 wave + 8 jj + 4 hh ..: what lane half hh of the second product takes
    // as its jj-th half.
    const int key = tid >> 2, e = tid & 3;
    const int jj = tid & 1, word = tid >> 1 & 15, hh = tid >> 5 & 1, piece = 2 * wave + hh;
    const int first_of_four = 8 * jj + 4 * hh;             // of the wave's sixteen
    const uint32_t k_at = (uint32_t)((key & ~15) + (key >> 2 & 1) * 8 + (key >> 3 & 1) * 4 + (key & 3));      // the key's place in the order of the second product
    const uint32_t k_to = (uint32_t)(key * kKeyRow + e * 64);                 // piece 4 e + i of a key's row (fp16 pages: it holds dimensions 8 (e + 4 i) ..)
    const int v_row = 4 * (word & 1) + 8 * (word >> 1 & 1) + 32 * (word >> 2);              // row of dimension 8 word; 8 word + 4 is 16 rows on
    const uint32_t v_to = (uint32_t)(dim_row(v_row) + jj * 8 + piece * 16);

    for (int r_tile = tile * kRows;; r_tile += a.tiles * kRows) {
        int first_step = 0, end_step = 0;
        if (DEALT) {
            const int tile_steps = len > 0 ? ((len - 1) >> 6) + 1 : 1;         // (of an empty prefix: one that shows nothing)
            const int64_t tiles = (int64_t)c.num_heads * a.tiles;
            const int shares = dealt_shares(tiles, tile_steps, a.dealt), eighths = shares >> 3;
            const int share = (int)blockIdx.x < eighths * 8 ? (int)(blockIdx.x & 7) * eighths + (int)(blockIdx.x >> 3) : (int)blockIdx.x;
            DealtPiece piece;
            if (!dealt_piece(tiles, tile_steps, shares, share, done, piece)) break;
            first_step = piece.first, end_step = piece.end, split = piece.state;
            head = piece.tile / a.tiles, r_tile = (piece.tile - head * a.tiles) * kRows;
            head_slots = ((int64_t)c.layer_idx * 2 * c.num_heads + head) * c.page_size;
            done += end_step - first_step;
            if (r_tile >= rows) continue;
        } else if (r_tile >= rows) {
            break;
        }
        const int r_end = r_tile + kRows < rows ? r_tile + kRows : rows;
        const int tile_lowest = first_place + divided(r_tile, a.per_place), tile_highest = first_place + divided(r_end - 1, a.per_place);
        const Steps steps = steps_of<6>(a, tile_lowest, tile_highest);
        const int s_begin = DEALT ? first_step : divided(steps.all * split, a.per_split);      // (below 2^24 steps, 2^5 splits)
        const int s_end = DEALT ? (end_step < steps.all ? end_step : steps.all) : divided(steps.all * (split + 1), a.per_split);
        const int last = s_end - 1;
        auto position = [&](int s) INLINE { return steps.at(s < last ? s : last) * kStep; };        // (behind the last step the last again)

        // ALIGNED: page numbers of the wave's sixteen positions in the next 64 steps, a lane each, -1: none; a step takes its own by a lane's number
        int page64 = -1, page64_from = 0;
        auto ask_pages = [&](int s, int& it) INLINE {
            it = divided(position(s + lane) + 16 * wave, pages);
            return npages > 0 ? c.indices[p0 + (it < npages ? it : 0)] : -1;
        };
        auto fetch_pages = [&](int s) INLINE {
            int it;
            const int page = ask_pages(s, it);
            page64 = it < npages && page < c.num_pages ? page : -1;
            page64_from = s;
        };
        auto slot_of_lane = [&](int pos, bool& there) INLINE {    // pages of any size: every lane for itself
            const int it = divided(pos, pages);
            const u32 entry = (u32)(pos - it * c.page_size);
            const bool inside = pos < len && it < npages && entry < (u32)c.page_size;
            const int page = npages > 0 ? c.indices[p0 + (inside ? it : 0)] : -1;
            there = inside && page >= 0 && page < c.num_pages;
            return there ? page * page_slots + head_slots + entry : head_slots;
        };
        // slot of the first of the wave's sixteen positions (of page 0 where they are not there; pages of any size: of the lane's own, the first sixteen lanes') and
        // which of them are there
        struct Sixteen {
            int64_t slot;
            u32 mask;
        };
        auto sixteen_of = [&](int s) INLINE {
            const int at = position(s) + 16 * wave;
            if (!ALIGNED) {
                bool there;
                const int64_t slot = slot_of_lane(at + (lane & 15), there);
                return Sixteen{slot, (u32)__builtin_amdgcn_ballot_w64(there) & 0xFFFFu};
            }
            const int page = __builtin_amdgcn_readlane(page64, (s < last ? s : last) - page64_from & 63);
            const u32 entry = (u32)(at - divided(at, pages) * c.page_size);
            const bool there = page >= 0 && entry < (u32)c.page_size;
            const int left = len - at;
            return Sixteen{there ? page * page_slots + head_slots + entry : head_slots, !there || left <= 0 ? 0u : left >= 16 ? 0xFFFFu : (1u << left) - 1u};
        };
        auto mask_of = [&](bool there) INLINE {                   // of a bool that the four lanes of a key share
            const uint64_t lanes = __builtin_amdgcn_ballot_w64(there);
            u32 mask = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) mask |= (u32)(lanes >> (4 * i) & 1) << i;
            return mask;
        };
        auto fetch_keys = [&](KeyCodes<F16>& f, const Sixteen& all) INLINE {
            if (ALIGNED) {
                const int64_t base = all.slot;
                f.mask = all.mask;
                const uint8_t* const kd = c.data + base * VEC;
                uint32_t off = (uint32_t)(lane >> 2) * VEC + (uint32_t)e * 16, p_off = (uint32_t)(lane >> 2) * 4;
                asm volatile("" : "+v"(off), "+v"(p_off));                         // (32-bit offsets behind wave-uniform addresses)
#pragma unroll
                for (int i = 0; i < (F16 ? 4 : 1); ++i) f.k[i] = *(const u32x4*)(kd + off + 64 * i);
                if (!F16) {
                    f.p = *(const u32*)((const uint8_t*)(c.param + base) + p_off);
                    f.pv = *(const u32*)((const uint8_t*)(c.param + base + kv_slots) + p_off);
                }
            } else {
                const int64_t base = __shfl(all.slot, lane >> 2, 64);
                f.mask = all.mask;
                const uint8_t* const kd = c.data + base * VEC + e * 16;
#pragma unroll
                for (int i = 0; i < (F16 ? 4 : 1); ++i) f.k[i] = *(const u32x4*)(kd + 64 * i);
                if (!F16) f.p = c.param[base], f.pv = c.param[base + kv_slots];
            }
        };
        auto fetch_values = [&](ValueCodes<F16>& f, const Sixteen& all) INLINE {
            if (ALIGNED) {
                const int64_t base = all.slot + kv_slots;
                f.mask = all.mask;
                const uint8_t* const vd = c.data + base * VEC;
                const uint8_t* const vp = (const uint8_t*)(c.param + base);
                uint32_t off = (uint32_t)first_of_four * VEC + (uint32_t)word * (VEC / 16), p_off = (uint32_t)first_of_four * 4, own = (uint32_t)(lane >> 2) * 4;
                asm volatile("" : "+v"(off), "+v"(p_off), "+v"(own));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (F16) f.v4[i] = *(const u32x4*)(vd + off + VEC * i);
                    else f.v[i] = *(const u32*)(vd + off + VEC * i), f.scales[i] = *(const u32*)(vp + p_off + 4 * i);
                }
                if (!F16) f.p = *(const u32*)(vp + own);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int64_t slot = __shfl(all.slot, first_of_four + i, 64) + kv_slots;
                    const uint8_t* const vd = c.data + slot * VEC + word * (VEC / 16);
                    if (F16) f.v4[i] = *(const u32x4*)vd;
                    else f.v[i] = *(const u32*)vd, f.scales[i] = c.param[slot];
                }
                f.mask = all.mask;
                if (!F16) f.p = c.param[__shfl(all.slot, lane >> 2, 64) + kv_slots];
            }
        };
        // pieces of the unpacking, small enough to stand between matrix instructions; kbuf, vbuf: offsets in LDS
        auto place_key = [&](const KeyCodes<F16>& f, uint32_t kbuf, int i) INLINE {
            *(u32x4*)(lds + (k_to + kbuf) + 16 * i) = F16 ? f.k[F16 ? i : 0] : codes_of(f.k[0][i]);
        };
        struct KeyLine {                                   // a key's slope and what the logits' line has of it: zero point, log2 of its value's factor
            float slope;
            u32x4 lower;
            u32x2 upper;
        };
        auto key_line = [&](const KeyCodes<F16>& f) INLINE {
            KeyLine l;
            if (F16) return l;
            const f16x2 p = as_f16x2(f.p);
            const float zero = (float)p[1], zero_hi = top(zero), zero_lo = zero - zero_hi;
            const u32 hi2 = tops(zero_hi, zero_hi), lo2 = tops(zero_lo, zero_lo);
            const float scale = __builtin_fabsf((float)as_f16x2(f.pv)[0]), log = __builtin_amdgcn_logf(factor_of(scale, power_of(scale)));
            const float l1 = top(log), l2 = top(log - l1), l3 = log - l1 - l2;
            l.slope = (float)p[0] * (kLog2e * kScale * kCodeUnit);
            l.lower = u32x4{hi2, tops(zero_hi, zero_lo), lo2, 0x3F803F80u};
            l.upper = u32x2{tops(1.f, l1), tops(l2, l3)};
            return l;
        };
        auto place_key_line = [&](const KeyCodes<F16>& f, const KeyLine& l, uint32_t kbuf) INLINE {
            if (e == 0) {
                if (!F16) {
                    *(float*)(lds + (kbuf + kSlope + k_at * 4)) = l.slope;
                    *(u32x4*)(lds + (kbuf + kLine + (uint32_t)key * 16)) = l.lower;
                    *(u32x2*)(lds + (kbuf + kLine + 1024 + (uint32_t)key * 16)) = l.upper;
                }
                if (lane == 0) *(unsigned short*)(lds + (kbuf + kThere + 2 * wave)) = (unsigned short)f.mask;
            }
        };
        auto store_values = [&](uint32_t vbuf, int half, const u32 (&out)[4][2]) INLINE {             // rows v_row + 16 half + i
#pragma unroll
            for (int i = 0; i < 4; ++i) *(u32x2*)(lds + (v_to + vbuf) + (16 * half + i) * kDimRow) = u32x2{out[i][0], out[i][1]};
        };
        auto place_value = [&](const ValueCodes<F16>& f, uint32_t vbuf, int half, const u32* power) INLINE {         // dimensions 8 word + 4 half ..
            u32 out[4][2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (F16) {
                    const u32x4 x = f.v4[F16 ? 2 * k : 0], y = f.v4[F16 ? 2 * k + 1 : 0];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        out[2 * i][k] = __builtin_amdgcn_perm(y[2 * half + i], x[2 * half + i], 0x05040100u);
                        out[2 * i + 1][k] = __builtin_amdgcn_perm(y[2 * half + i], x[2 * half + i], 0x07060302u);
                    }
                } else {
                    const u32x4 w = scaled_codes(__builtin_amdgcn_perm(f.v[F16 ? 0 : 2 * k + 1], f.v[F16 ? 0 : 2 * k], half ? 0x07060302u : 0x05040100u), power[k]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[i][k] = w[i];
                }
            }
            store_values(vbuf, half, out);
        };
        auto place_value_half = [&](const ValueCodes<F16>& f, uint32_t vbuf, int half, int cb, const u32* power) INLINE {
            if (cb == 1) place_value(f, vbuf, half, power);
        };
        auto place_value_parameters = [&](u32 p, u32 odd, uint32_t vbuf) INLINE {                     // p: of the position with the key's number
            if (!F16) {
                const f16x2 v = as_f16x2(p);
                const float scale = __builtin_fabsf((float)v[0]), recip = __builtin_amdgcn_rcpf(factor_of(scale, power_of(scale))), zero = (float)v[1] * recip;
                const f16 recip_hi = (f16)recip, zero_hi = (f16)zero, recip_lo = (f16)((recip - (float)recip_hi) * 2048.f), zero_lo = (f16)((zero - (float)zero_hi) * 2048.f);
                if (e == 0) {
                    uint8_t* const extra_rows = lds + (vbuf + dim_row(128) + k_at * 2);
                    *(f16*)extra_rows = recip_hi, *(f16*)(extra_rows + kDimRow) = recip_lo;
                    *(f16*)(extra_rows + 2 * kDimRow) = zero_hi, *(f16*)(extra_rows + 3 * kDimRow) = zero_lo;
                }
            }
            if (lane == 0) *(unsigned short*)(lds + (vbuf + kOdd + 2 * wave)) = (unsigned short)odd;
        };
        // 2^e of the four positions' scales in pairs (a negative scale's sign is its power's: not plain); whether the short way is right for all of the wave's positions (fp16 pages: only where all of the tile's
        // rows see them)
        auto regular = [&](const ValueCodes<F16>& f, u32* power, bool all_see) INLINE {
            if (F16) return f.mask == 0xFFFFu && all_see;
            bool plain = !strange(f.p) && !(f.p & 0x8000u);
#pragma unroll
            for (int k = 0; k < 2; ++k) power[k] = powers_of(f.scales[F16 ? 0 : 2 * k], f.scales[F16 ? 0 : 2 * k + 1], plain);
            return f.mask == 0xFFFFu && __builtin_amdgcn_ballot_w64(!plain) == 0;
        };
        // any values: positions that are not there count as zero, those whose parameters are not finite (fp16 pages: their entries that are not) as well, and are
        // marked
        auto place_values_any = [&](const ValueCodes<F16>& f, uint32_t vbuf) INLINE {
            auto there = [&](int i) { return (f.mask >> (first_of_four + i) & 1) != 0; };
            if (F16) {
                ValueCodes<F16> g = f;
                u32 odd = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bool any = false;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const u32 w = there(i) ? (u32)f.v4[F16 ? i : 0][j] : 0u;
                        any = any || strange(w);
                        g.v4[F16 ? i : 0][j] = ((w & 0x7C00u) == 0x7C00u ? 0u : w & 0xFFFFu) | ((w & 0x7C000000u) == 0x7C000000u ? 0u : w & 0xFFFF0000u);
                    }
                    const uint64_t lanes = __builtin_amdgcn_ballot_w64(any);
                    odd |= ((lanes & 0x55555555u) ? 1u << i : 0) | ((lanes & 0xAAAAAAAAu) ? 1u << (8 + i) : 0);
                    odd |= ((lanes >> 32 & 0x55555555u) ? 1u << (4 + i) : 0) | ((lanes >> 32 & 0xAAAAAAAAu) ? 1u << (12 + i) : 0);
                }
                place_value_parameters(0, odd, vbuf);
#pragma unroll
                for (int half = 0; half < 2; ++half) place_value(g, vbuf, half, nullptr);
            } else {
                u32 p[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) p[i] = !there(i) || strange(f.scales[F16 ? 0 : i]) ? kNoParameters : f.scales[F16 ? 0 : i];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    u32 out[4][2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const u32x4 w = scaled_codes_slow(__builtin_amdgcn_perm(f.v[F16 ? 0 : 2 * k + 1], f.v[F16 ? 0 : 2 * k], half ? 0x07060302u : 0x05040100u), p[2 * k], p[2 * k + 1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) out[i][k] = w[i] ^ (p[2 * k] & 0x8000u) ^ (p[2 * k + 1] & 0x8000u) << 16;
                    }
                    store_values(vbuf, half, out);
                }
                const bool mine = (f.mask >> (lane >> 2) & 1) != 0, odd = mine && strange(f.p);
                place_value_parameters(mine && !odd ? f.p : kNoParameters, mask_of(odd), vbuf);
            }
        };

        // the wave's rows: block cb has rows r0 + 32 cb + n
        const int r0 = r_tile + 64 * wave;
        const int r_last = r0 + 63 < rows ? r0 + 63 : rows - 1;
        // (a wave without rows hides nothing: its results go nowhere, and the others wait for it)
        const int lowest = r0 < rows ? first_place + divided(r0, a.per_place) : 0x7fffffff, highest = r0 < rows ? first_place + divided(r_last, a.per_place) : -1;
        auto row_of = [&](int cb) { return r0 + 32 * cb + n; };
        auto token_of = [&](int cb) { return divided(row_of(cb) < rows ? row_of(cb) : r_tile, a.per_group); };
        auto head_of = [&](int cb, int token) { return head * a.group + (row_of(cb) < rows ? row_of(cb) : r_tile) - token * a.group; };
        int place[2];

        // the queries: lane (n, h) holds piece 2 s + h of its rows, dimensions 16 s + 8 h .. + 7 (fp16 pages: in the order of k_to)
        int first_it = 0, first_page = -1;                 // (asked for ahead of the queries, taken behind them)
        if (ALIGNED && s_begin < s_end) first_page = ask_pages(s_begin, first_it);
        u32x4 qf[2][8], line[2];                           // line: the logits' line, {-zero-point slope in three pieces, twice; the maximum's}
        float slope[2];
#pragma unroll
        for (int cb = 0; cb < 2; ++cb) {
            const bool in = row_of(cb) < rows;
            const int token = token_of(cb);
            place[cb] = in ? first_place + divided(row_of(cb), a.per_place) : -1;
            const u32x4* src = (const u32x4*)(a.q + (int64_t)(tokens.start + token) * a.q_stride + (int64_t)head_of(cb, token) * 128) + (F16 ? 4 * h : h);
#pragma unroll
            for (int s = 0; s < 8; ++s) qf[cb][s] = src[F16 ? (s >> 1) + 8 * (s & 1) : 2 * s];       // (rows that are not there: another one's, whose results go nowhere)
        }
        KeyCodes<F16> fk, fk1;
        ValueCodes<F16> fv;
        Sixteen all0{}, all1{}, all2{};                    // of this step, the next one and the one behind it
        if (s_begin < s_end) {
            page64 = first_it < npages && first_page < c.num_pages ? first_page : -1, page64_from = s_begin;
            all0 = sixteen_of(s_begin), all1 = sixteen_of(s_begin + 1), all2 = sixteen_of(s_begin + 2);
            fetch_keys(fk, all0);
            fetch_values(fv, all0);
            fetch_keys(fk1, all1);
        }
        __syncthreads();                                   // (what never changes; the last tile's buffers)

#pragma unroll
        for (int cb = 0; cb < 2; ++cb) {
            if (__builtin_expect(a.q_had, 0)) {
                float v[64];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const f16x2 p = as_f16x2(qf[cb][i >> 2][i & 3]);
                    v[2 * i] = (float)p[0], v[2 * i + 1] = (float)p[1];
                }
#pragma unroll
                for (int bit = 1; bit < 64; bit *= 2)
#pragma unroll
                    for (int i = 0; i < 64; ++i)
                        if (!(i & bit)) {
                            const float x = v[i], y = v[i | bit];
                            v[i] = x + y, v[i | bit] = x - y;
                        }
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                    const u32x2 w = both_halves<32>(as_u32(v[i]));
                    v[i] = h ? as_f32(w.x) - as_f32(w.y) : as_f32(w.x) + as_f32(w.y);
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) qf[cb][i >> 2][i & 3] = narrow_f16x2(v[2 * i] * kScale, v[2 * i + 1] * kScale);
            }
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const f16x2 p = as_f16x2(qf[cb][i >> 2][i & 3]);
                sum += (float)p[0] + (float)p[1];
            }
            const u32x2 w = both_halves<32>(as_u32(sum));
            slope[cb] = (as_f32(w.x) + as_f32(w.y)) * -(kLog2e * kScale);
            if (!F16) {
#pragma unroll
                for (int s = 0; s < 8; ++s) qf[cb][s] = query_for_codes(qf[cb][s]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) asm volatile("" : "+a"(qf[0][i]), "+a"(qf[1][i]));       // (where they stay)
        float most[2] = {0.f, 0.f}, m[2] = {0.f, 0.f}, limit[2] = {-3e38f, -3e38f}, poison[2] = {0.f, 0.f};         // limit: until a row has seen a position, any logit moves its maximum
        auto draw_line = [&](int cb) INLINE {                     // lane half 0: slope pieces 1 2 3, 1 2 3, maximum pieces 1 2; half 1: piece 3, and ones
            const float s1 = top(slope[cb]), s2 = top(slope[cb] - s1), s3 = slope[cb] - s1 - s2;
            const float m1 = top(-m[cb]), m2 = top(-m[cb] - m1), m3 = -m[cb] - m1 - m2;
            const u32x4 lower = {tops(s1, s2), tops(s3, s1), tops(s2, s3), tops(m1, m2)}, upper = {tops(m3, 1.f), 0x3F803F80u, 0, 0};
            line[cb] = h ? upper : lower;
        };
        draw_line(0), draw_line(1);

        f32x16 acc[2][4], extra[2], x[2], y[2];            // y: the logits of the unit at work, then x those of the next
#pragma unroll
        for (int cb = 0; cb < 2; ++cb) acc[cb][0] = acc[cb][1] = acc[cb][2] = acc[cb][3] = extra[cb] = zeros();
        u32x4 p[2][2];                                     // weights: [rows][half unit]

        const uint32_t k_from = n * kKeyRow + h * 16, v_from = dim_row(n) + h * 16;
        const uint32_t e_from = dim_row(128) + (n < 4 ? n : 4) * kDimRow + h * 16, l_from = kLine + h * 1024 + n * 16, s_from = kSlope + h * 32;
        auto key_piece = [&](uint32_t kbuf, int kb, int i) INLINE { return *(const u32x4*)(lds + (k_from + kbuf) + kb * 32 * kKeyRow + i * 32); };
        auto value_piece = [&](uint32_t vbuf, int chunk, int db) INLINE {
            return db < 4 ? *(const u32x4*)(lds + (v_from + vbuf) + dim_row(32 * db) + chunk * 32) : *(const u32x4*)(lds + (e_from + vbuf) + chunk * 32);
        };

        // row of block cb: sees positions up to its place, from behind `before` on, and the sinks
        auto before = [&](int cb) INLINE { return a.window ? place[cb] - a.window : -1; };
        auto sees = [&](int cb, int pos) INLINE { return (pos <= place[cb]) & ((pos > before(cb)) | (pos < a.sinks)); };
        // Of the next unit: whether its positions are all there and all seen (`at`: its first); else the logits that are not seen are taken out
        u32 there = 0;
        auto all_seen = [&](int at) INLINE { return at + 31 <= lowest && (a.window == 0 || at > highest - a.window || at + 31 < a.sinks); };
        // (most units that are not all seen lie on one edge only: of the diagonal, or of the window)
        auto hide = [&](int at) INLINE {
            const u32 all = __builtin_amdgcn_readfirstlane(there);
            const bool all_begun = a.window == 0 || at > highest - a.window, all_ended = at + 31 <= lowest && at >= a.sinks;
#pragma unroll
            for (int cb = 0; cb < 2; ++cb) {
                const int from = at + 4 * h, high = place[cb] - from, low = before(cb) - from, sinks = a.sinks - from;
                most[cb] = -__builtin_inff();
                if (all_begun) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[cb][i] = 8 * (i >> 2) + (i & 3) <= high ? y[cb][i] : -__builtin_inff();
                } else if (all_ended) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[cb][i] = 8 * (i >> 2) + (i & 3) > low ? y[cb][i] : -__builtin_inff();
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int k = 8 * (i >> 2) + (i & 3);
                        y[cb][i] = (k <= high) & ((k > low) | (k < sinks)) ? y[cb][i] : -__builtin_inff();
                    }
                }
                if (~all) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) y[cb][i] = all >> (8 * (i >> 2) + 4 * h + (i & 3)) & 1 ? y[cb][i] : -__builtin_inff();
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) most[cb] = __builtin_fmaxf(most[cb], y[cb][i]);
            }
        };
        // Marked positions of the unit at work.  Int4 pages: rows that see one become NaN.  Fp16 pages: its entries that are not finite are added for the rows that
        // see it, by a product of bf16 powers of two that overflows to an infinity (a NaN: to one of each sign).
        u32 odd = 0;
        auto mark = [&](int at) INLINE {
            const u32 bits = __builtin_amdgcn_readfirstlane(odd);
            if (bits != 0) {
#pragma unroll 1
                for (int k = 0; k < 32; ++k) {
                    if (!(bits >> k & 1)) continue;
                    if (!F16) {
                        poison[0] = sees(0, at + k) ? __builtin_nanf("") : poison[0];
                        poison[1] = sees(1, at + k) ? __builtin_nanf("") : poison[1];
                        continue;
                    }
                    bool there;
                    const unsigned short* const v = (const unsigned short*)(c.data + (slot_of_lane(at + k, there) + kv_slots) * VEC) + 8 * (n >> 2 & 3) + 4 * (n >> 4) + (n & 3);
                    const u32x4 seen[2] = {{h == 0 && sees(0, at + k) ? 0x7F00u : 0u, 0, 0, 0}, {h == 0 && sees(1, at + k) ? 0x7F00u : 0u, 0, 0, 0}};
#pragma unroll
                    for (int db = 0; db < 4; ++db) {
                        const u32 bf = v[32 * db], sign = bf & 0x8000u;
                        const bool nan = (bf & 0x7FFFu) > 0x7C00u, inf = (bf & 0x7FFFu) == 0x7C00u;
                        const u32x4 up = {h == 0 && (nan || (inf && !sign)) ? 0x7F00u : 0u, 0, 0, 0}, down = {h == 0 && (nan || (inf && sign)) ? 0xFF00u : 0u, 0, 0, 0};
#pragma unroll
                        for (int cb = 0; cb < 2; ++cb) {
                            mfma_overflow(acc[cb][db], up, seen[cb]);
                            mfma_overflow(acc[cb][db], down, seen[cb]);
                        }
                    }
                }
            }
        };
        auto begin = [&]() INLINE {                         // the first maxima
#pragma unroll
            for (int cb = 0; cb < 2; ++cb) {
                const u32x2 both = both_halves<32>(as_u32(most[cb]));
                const float now = __builtin_fmaxf(as_f32(both.x), as_f32(both.y));
                const bool any = now > limit[cb];
                m[cb] = any ? now - kBase : 0.f, most[cb] -= m[cb];
                limit[cb] = any ? kHigh : limit[cb];
#pragma unroll
                for (int i = 0; i < 16; ++i) y[cb][i] -= m[cb];
                draw_line(cb);
            }
        };
        auto raise = [&]() INLINE {
#pragma unroll
            for (int cb = 0; cb < 2; ++cb) {
                const u32x2 both = both_halves<32>(as_u32(most[cb]));
                const float now = __builtin_fmaxf(as_f32(both.x), as_f32(both.y));
                const bool moves = now > limit[cb];        // (of the row alone: what other rows see changes nothing)
                // (nothing seen so far: the sums are zero, and a first maximum far below zero would make them zero times an infinity)
                const float by = moves ? now - kBase : 0.f, keep = limit[cb] < 0.f ? 0.f : __builtin_amdgcn_exp2f(-by);
                limit[cb] = moves ? kHigh : limit[cb];
                m[cb] += by;
#pragma unroll
                for (int i = 0; i < 16; ++i) y[cb][i] -= by;
#pragma unroll
                for (int k = 0; k < 5; ++k) {
                    f32x16& block = k < 4 ? acc[cb][k & 3] : extra[cb];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float v = block[i];
                        scale_accumulator(v, keep);
                        block[i] = v;
                    }
                }
                draw_line(cb);
            }
        };
        // two weights (times the values' factors, which are in the logits) of half unit tt: registers 8 tt + 2 j, + 1
        auto weights = [&](const f32x16& v, int tt, int j) INLINE {
            return cvt_f16x2(__builtin_amdgcn_exp2f(v[8 * tt + 2 * j]), __builtin_amdgcn_exp2f(v[8 * tt + 2 * j + 1]));
        };
        auto weigh = [&]() INLINE {
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i >> 3][i >> 2 & 1][i & 3] = weights(y[i >> 3], i >> 2 & 1, i & 3);
        };
        // First product of unit kb of the keys at kbuf into x; between it the weights of the unit at work, unit `unit` of the values at vbuf, and whether one of
        // its maxima has to be raised (which makes the weights anew).  Operands come from LDS three slots ahead.
        u32x4 kp[3], vp[3], ln;
        f32x4 slopes[4];
        bool grow = false;
        auto ask_keys = [&](uint32_t kbuf, int kb) INLINE {
#pragma unroll
            for (int i = 0; i < 3; ++i) kp[i] = key_piece(kbuf, kb, i);
        };
        auto ask_line = [&](uint32_t kbuf, int kb) INLINE {
            if (F16) return;
            ln = *(const u32x4*)(lds + (l_from + kbuf) + kb * 512);
#pragma unroll
            for (int i = 0; i < 4; ++i) slopes[i] = *(const f32x4*)(lds + (s_from + kbuf) + kb * 128 + (i >> 1) * 64 + (i & 1) * 16);
        };
        auto first_product = [&](uint32_t kbuf, int kb, uint32_t vbuf, int unit, bool with_weights, auto&& other) INLINE {
            float ahead[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) {
                    if (i == 0) mfma_first(x[cb], kp[i % 3], qf[cb][i]);
                    else mfma_more(x[cb], kp[i % 3], qf[cb][i]);
                    if (with_weights) {
                        // (a pair's exponentials in one slot, their conversion in the next; here, not behind the question whether they are made anew)
                        float w0 = __builtin_amdgcn_exp2f(y[cb][2 * i]), w1 = __builtin_amdgcn_exp2f(y[cb][2 * i + 1]);
                        if (i + cb > 0) {
                            const int j = cb ? i : i - 1;
                            u32 w = cvt_f16x2(ahead[0], ahead[1]);
                            asm volatile("" : "+v"(w));
                            p[cb ^ 1][j >> 2][j & 3] = w;
                        }
                        asm volatile("" : "+v"(w0), "+v"(w1));
                        ahead[0] = w0, ahead[1] = w1;
                        if (cb == 0 && i == 1) grow = __builtin_amdgcn_ballot_w64(most[0] > limit[0] || most[1] > limit[1]) != 0;
                    }
                    if (cb == 0) other(i);
                    if (cb == 1 && i < 5) kp[i % 3] = key_piece(kbuf, kb, i + 3);
                    if (cb == 1 && i == 5) ask_line(kbuf, kb);
                    if (cb == 0 && i > 4) vp[i - 5] = value_piece(vbuf, 2 * unit, i - 5);
                    SLOT;
                }
            }
            if (with_weights) p[1][1][3] = cvt_f16x2(ahead[0], ahead[1]);
        };
        // Second product of the unit at work; between it the logits of the next one, unit next_kb of the keys at kbuf, from its first product and their line,
        // and their maxima.
        auto second_product = [&](uint32_t vbuf, int unit, uint32_t kbuf, int next_kb, auto&& other) INLINE {
            if (!F16) {
                mfma_line(y[0], ln, line[0]);
                mfma_line(y[1], ln, line[1]);
                SLOT;
            }
            there = *(const u32*)(lds + (kbuf + kThere) + 4 * next_kb);
            odd = *(const u32*)(lds + (vbuf + kOdd) + 4 * unit);
#pragma unroll
            for (int i = 0; i < 10; ++i) {
                const int tt = i / 5, db = i % 5;
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) {
                    mfma_second(db < 4 ? acc[cb][db & 3] : extra[cb], vp[i % 3], p[cb][tt]);
                    if (i > 1) {
                        const int reg = 2 * (i - 2);
                        float y0 = F16 ? __builtin_fmaf(x[cb][reg], kLog2e * kScale, -m[cb]) : __builtin_fmaf(x[cb][reg], slopes[reg >> 2][reg & 3], y[cb][reg]);
                        float y1 = F16 ? __builtin_fmaf(x[cb][reg + 1], kLog2e * kScale, -m[cb]) : __builtin_fmaf(x[cb][reg + 1], slopes[reg >> 2][(reg & 3) + 1], y[cb][reg + 1]);
                        most[cb] = i == 2 ? __builtin_fmaxf(y0, y1) : __builtin_fmaxf(__builtin_fmaxf(most[cb], y0), y1);
                        asm volatile("" : "+v"(y0), "+v"(y1), "+v"(most[cb]));         // (here, not where they are used)
                        y[cb][reg] = y0, y[cb][reg + 1] = y1;
                    }
                    if (cb == 1 && i < 7) vp[i % 3] = value_piece(vbuf, 2 * unit + (i + 3) / 5, (i + 3) % 5);
                    other(i, cb);
                    SLOT;
                }
            }
        };

        // offsets in LDS: this step's keys, the next one's and those of the step behind it; this step's values and the next one's
        uint32_t k0 = 0, k1 = kKeys, k2 = 2 * kKeys, v0 = 3 * kKeys, v1 = 3 * kKeys + kValues;
        int s = s_begin;
        if (s_begin < s_end) {
#pragma unroll
            for (int i = 0; i < 4; ++i) place_key(fk, k0, i);
            place_key_line(fk, key_line(fk), k0);
            u32 power[2];
            if (!F16 && regular(fv, power, true)) {
                place_value(fv, v0, 0, power);
                place_value(fv, v0, 1, power);
                place_value_parameters(fv.p, 0, v0);
            } else {
                place_values_any(fv, v0);
            }
            fetch_keys(fk, all2);
#pragma unroll
            for (int i = 0; i < 4; ++i) place_key(fk1, k1, i);
            place_key_line(fk1, key_line(fk1), k1);
        }
        __syncthreads();
        if (s_begin < s_end) {
            ask_keys(k0, 0);
            first_product(k0, 0, v0, 0, false, [](int) {});
            f32x16 t[2];
            if (!F16) {
                mfma_line(t[0], ln, line[0]);
                mfma_line(t[1], ln, line[1]);
            }
            there = *(const u32*)(lds + k0 + kThere);
            settled();
#pragma unroll
            for (int cb = 0; cb < 2; ++cb)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    y[cb][i] = F16 ? __builtin_fmaf(x[cb][i], kLog2e * kScale, -m[cb]) : __builtin_fmaf(x[cb][i], slopes[i >> 2][i & 3], t[cb][i]);
            if (!F16 && all_seen(position(s_begin)) && ~__builtin_amdgcn_readfirstlane(there) == 0) {
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) {
                    most[cb] = y[cb][0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) most[cb] = __builtin_fmaxf(most[cb], y[cb][i]);
                }
            } else {
                hide(position(s_begin));
            }
            begin();
            ask_keys(k0, 1);
        }
        // Units of 32 positions, two to a step.  (A wave whose rows see none of them goes through them all the same: it would wait for the others.)
        auto first_of_0 = [&]() INLINE {                   // weights of unit 0, first product of unit 1
            first_product(k0, 1, v0, 0, true, [&](int i) {
                if (i == 2) fetch_values(fv, all1);
            });
        };
        auto second_of_0 = [&]() INLINE {
            bool usual = false;
            KeyLine l;
            const int at = position(s);
            second_product(v0, 0, k0, 1, [&](int i, int cb) {
                if (i < 2) place_key(fk, k2, 2 * i + cb);
                if (i == 4 && cb == 0) l = key_line(fk);
                if (i == 6 && cb == 0) place_key_line(fk, l, k2);
                if (i == 8 && cb == 0) usual = all_seen(at + 32) && (~__builtin_amdgcn_readfirstlane(there) | __builtin_amdgcn_readfirstlane(odd)) == 0;
                if (i == 9 && cb == 1) ask_keys(k1, 0);
            });
            if (__builtin_expect(!usual, 0)) mark(at), hide(at + 32);
        };
        auto first_of_1 = [&]() INLINE {
            all0 = all1, all1 = all2, all2 = sixteen_of(s + 3);
            first_product(k1, 0, v0, 1, true, [&](int i) {
                if (i == 2) fetch_keys(fk, all2);
            });
        };
        auto second_of_1 = [&]() INLINE {
            u32 power[2];
            bool usual = false;
            const int at = position(s), next = position(s + 1);
            const bool regular_values = regular(fv, power, next + 63 <= tile_lowest && (a.window == 0 || next > tile_highest - a.window || next + 63 < a.sinks));
            second_product(v0, 1, k1, 0, [&](int i, int cb) {
                if (i == 0 || i == 3) place_value_half(fv, v1, i == 3, cb, power);
                if (i == 6 && cb == 0) place_value_parameters(fv.p, 0, v1);
                if (i == 8 && cb == 0) usual = all_seen(next) && (~__builtin_amdgcn_readfirstlane(there) | __builtin_amdgcn_readfirstlane(odd)) == 0;
                if (i == 9 && cb == 1) ask_keys(k1, 1);
            });
            if (__builtin_expect(!regular_values, 0)) place_values_any(fv, v1);
            if (__builtin_expect(!usual, 0)) mark(at + 32), hide(next);
            ++s;
            if (ALIGNED && __builtin_expect(s + 3 - page64_from >= 64, 0)) fetch_pages(s);
            __syncthreads();
            const uint32_t k = k0, v = v0;
            k0 = k1, k1 = k2, k2 = k, v0 = v1, v1 = v;
        };
        auto raised = [&]() INLINE {
            settled();
            raise();
            weigh();
        };
        while (s < s_end) {
            first_of_0();
            if (__builtin_expect(grow, 0)) raised();
            second_of_0();
            first_of_1();
            if (__builtin_expect(grow, 0)) raised();
            second_of_1();
        }

        settled();
        // rows 0 .. 3 of the extra block, in the registers of the lower half: sums of weights (as pairs) and of weights times zero points
#pragma unroll
        for (int cb = 0; cb < 2; ++cb) {
            float sum = F16 ? extra[cb][0] : __builtin_fmaf(extra[cb][1], 1.f / 2048.f, extra[cb][0]);
            float zero = F16 ? 0.f : __builtin_fmaf(extra[cb][3], 1.f / 2048.f, extra[cb][2]);
            sum = as_f32(both_halves<32>(as_u32(sum)).x);
            if (!F16) {
                zero = as_f32(both_halves<32>(as_u32(zero)).x);
                const u32x2 both = both_halves<32>(as_u32(poison[cb]));
                sum += as_f32(both.x) + as_f32(both.y);
            }
            if (row_of(cb) >= rows) continue;
            const int token = token_of(cb), q_head = head_of(cb, token);
            // lane (n, h): dimensions 32 db + 16 i + 8 h + 4 k + j of row n in register 4 (i + 2 k) + j of block db
            if (!a.states) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum, less = -zero * inv;
                if (a.lse && h == 0) a.lse[(int64_t)(tokens.start + token) * (c.num_heads * a.group) + q_head] = lse_of(limit[cb] < 0.f ? kEmpty : m[cb], sum);
                u32x4* const dst = (u32x4*)(a.o + (int64_t)(tokens.start + token) * a.o_stride + (int64_t)q_head * 128) + h;
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        u32x4 w;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int reg = 4 * (i + 2 * (j >> 1)) + 2 * (j & 1);
                            w[j] = cvt_f16x2(__builtin_fmaf(acc[cb][db][reg], inv, less), __builtin_fmaf(acc[cb][db][reg + 1], inv, less));
                        }
                        dst[4 * db + 2 * i] = w;
                    }
            } else {
                float* const dst = a.part + (((int64_t)(tokens.start + token) * (c.num_heads * a.group) + q_head) * a.parts + a.part_at + split) * 132;
                if (h == 0) dst[0] = limit[cb] < 0.f ? kEmpty : m[cb], dst[1] = sum;
                if (DEALT && h == 0 && s_end == steps.all)
                    for (int i = a.part_at + split + 1; i < a.parts; ++i) dst[132 * (i - a.part_at - split)] = kEmpty, dst[132 * (i - a.part_at - split) + 1] = 0.f;
#pragma unroll
                for (int db = 0; db < 4; ++db)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *(f32x4*)(dst + 4 + 32 * db + 16 * (i & 1) + 8 * h + 4 * (i >> 1)) =
                            f32x4{acc[cb][db][4 * i] - zero, acc[cb][db][4 * i + 1] - zero, acc[cb][db][4 * i + 2] - zero, acc[cb][db][4 * i + 3] - zero};
            }
        }
    }
}

template <bool F16, bool ALIGNED>
__global__ __launch_bounds__(256, 1) void chunk_tiles_kernel(Chunk a, Divisor pages) { attend_tiles<F16, ALIGNED, false>(a, pages); }
// (a kernel of its own: what the shares need costs the other one registers, 4 % of its time on fp16 pages)
template <bool F16, bool ALIGNED>
__global__ __launch_bounds__(256, 1) void prefix_tiles_kernel(Chunk a, Divisor pages) { attend_tiles<F16, ALIGNED, true>(a, pages); }

}  // namespace

int qr_internal_chunk_tiles(bool fp16, const Chunk& a, Divisor pages, int64_t groups, hipStream_t st) {
    using Kernel = void (*)(Chunk, Divisor);
    const bool aligned = a.c.page_size % 16 == 0;
    const Kernel kernel = a.dealt ? (fp16 ? (aligned ? prefix_tiles_kernel<true, true> : prefix_tiles_kernel<true, false>)
                                          : (aligned ? prefix_tiles_kernel<false, true> : prefix_tiles_kernel<false, false>))
                          : fp16 ? (aligned ? chunk_tiles_kernel<true, true> : chunk_tiles_kernel<true, false>)
                               : (aligned ? chunk_tiles_kernel<false, true> : chunk_tiles_kernel<false, false>);
    const hipError_t e = qr_allow_dynamic_lds((const void*)kernel, kLds);
    if (e != hipSuccess) return (int)e;
    kernel<<<dim3((unsigned)groups), dim3(256), kLds, st>>>(a, pages);
    return qr_launch_status();
}
