// What attention gives to the cached positions, added up position by position, from the queries, the softmax's logarithmic sums and the keys:
//
//   W[b, h, j] += sum over the new tokens t of sequence b and the query heads g of key head h of exp( q[t, g] . k[j, h] / sqrt(128) - lse[t, g] )
//
// over the positions j that t sees (chunk.hip: all up to its own, or the last `window` and the first `sinks`).  A position belongs to one lane from
// its key to its sum: nothing is exchanged but the four partial sums of a column, no atomics, and the order of the additions is always the same.
//
// The logits are a product rows x positions, positions in the lanes: a position's scale and zero point are its lane's, sums over rows are sums of
// registers.  Int4 keys enter as codes, which fp16 holds exactly, q as it is.  Logits, exponentials and sums are in 32 bits, nothing is rounded to fewer.
#include "qr_chunk.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

namespace {

struct Weights {
    PagedKV c;
    const f16* q;
    const float* lse;
    float* sums;                      // [sequence, key head, capacity]
    const int32_t* starts;            // nullptr: one new token per sequence
    int64_t q_stride, capacity;
    int tokens, group, blocks, window, sinks, q_had;
    int64_t rows;                     // no sequence has more of a key head
    Divisor per_group, per_block, per_head;
    float* part;                      // splits > 1: sums of every split of the rows, [split, item, block, 256]
    int splits;
    uint8_t* units;                   // the queries as the kernel of many rows takes them: units of 32 rows, [key head, unit]
    int64_t all_units;
};

__device__ __forceinline__ Fresh fresh_of(const Weights& a, int b) {
    if (!a.starts) return Fresh{b, 1, 1};
    int start = a.starts[b];
    const int end = a.starts[b + 1];
    start = start < 0 ? 0 : start;
    const int stop = end > a.tokens ? a.tokens : end;
    return Fresh{start, stop > start ? stop - start : 0, end > start ? end - start : 0};
}

// The codes of a word as fp16 numbers, in the order of codes_of: (1024 + code) - 1024, (64 + code) - 64.  (As subnormal numbers, which codes_of makes without
// the subtraction, they lose bits on the way: a sum of 128 products is off by 27 steps of 2^-24 of itself then, root mean square, and by 0.6 like this, and
// the sums of 16384 rows by 2.4e-5 instead of 5e-7.)
__device__ __forceinline__ u32x4 numbers_of(u32 w, CodeMasks m) {
    const u32 w8 = w >> 8;
    const f16x2 a = {(f16)-1024.f, (f16)-1024.f}, b = {(f16)-64.f, (f16)-64.f};
    return u32x4{__builtin_bit_cast(u32, as_f16x2(and_or(w, m.low, 0x64006400u)) + a), __builtin_bit_cast(u32, as_f16x2(and_or(w, m.high, 0x54005400u)) + b),
                 __builtin_bit_cast(u32, as_f16x2(and_or(w8, m.low, 0x64006400u)) + a), __builtin_bit_cast(u32, as_f16x2(and_or(w8, m.high, 0x54005400u)) + b)};
}
// eight elements of q in the order of a word's codes: (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ u32x4 query_for_numbers(u32x4 w) {
    return u32x4{__builtin_amdgcn_perm(w[2], w[0], 0x05040100u), __builtin_amdgcn_perm(w[2], w[0], 0x07060302u),
                 __builtin_amdgcn_perm(w[3], w[1], 0x05040100u), __builtin_amdgcn_perm(w[3], w[1], 0x07060302u)};
}

// The Hadamard transform of a row whose 32 dimensions from 32 g on the lane (n, g) holds, rounded to fp16 like the transform's own entry point
__device__ __forceinline__ void hadamard_row(u32x4 (&w)[4], int lane) {
    float t32[32];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const f16x2 p = as_f16x2(w[i >> 2][i & 3]);
        t32[2 * i] = (float)p[0], t32[2 * i + 1] = (float)p[1];
    }
#pragma unroll
    for (int bit = 1; bit < 32; bit *= 2)
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (!(i & bit)) {
                const float x = t32[i], y = t32[i | bit];
                t32[i] = x + y, t32[i | bit] = x - y;
            }
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        u32x2 e = both_halves<16>(as_u32(t32[i]));
        const float v = (lane & 16) ? as_f32(e.x) - as_f32(e.y) : as_f32(e.x) + as_f32(e.y);
        e = both_halves<32>(as_u32(v));
        t32[i] = (lane & 32) ? as_f32(e.x) - as_f32(e.y) : as_f32(e.x) + as_f32(e.y);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i >> 2][i & 3] = narrow_f16x2(t32[2 * i] * kScale, t32[2 * i + 1] * kScale);
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------------
// A wave takes 64 positions of a (sequence, key head) at a time, lane by lane for their places, and all rows in tiles of 16: lane (n, g) holds quarter g of the
// keys of positions n, 16 + n, 32 + n and 48 + n.  While it works on them the next 64 positions' keys and sums are under way, and the page numbers of those behind.
// Of 16 rows and fewer the queries stay in registers, of up to 64 in LDS, ready for the products (a wave makes one tile of them; more are made for every block).
// One row and 32 heads after 3000: 5.0 us, a launch and one wave's chain of tables, pages, keys; 32 x one of 4001, 64 on 8 heads: 18.0 us, 4.4 TB/s of a copy's 5.2
// (every lane's loads of two blocks under way; half of the lanes without rows: 22.0); fp16 pages, 5 x up to 37 in a window of 1500, 40 heads: 15.6 us, 3.5 TB/s: 200 lists
// of unequal length, with as many workgroups each.
constexpr int kWaves = 4;
template <bool F16>
struct RowTile {                       // 16 rows: queries as the products take them; slope, logarithm (base 2, negative) and position of four of them
    u32x4 q[4];
    float slope[4] = {0.f, 0.f, 0.f, 0.f}, less[4];
    int place[4];
};
template <bool F16, bool HAD>
__device__ __forceinline__ RowTile<F16> row_tile(const Weights& a, const Fresh& mine, int h, int r0, int rows, int first_place, int lane, int quarter) {
    const int n = lane & 15, g = lane >> 4;                // quarter: which four rows' numbers the lane holds
    RowTile<F16> t;
    // lane (n, g) holds dimensions 32 g + 8 i .. (fp16 pages: 32 i + 8 g ..) of row n
    const int r = r0 + n < rows ? r0 + n : r0, token = divided(r, a.per_group), head = h * a.group + r - token * a.group;
    const u32x4* src = (const u32x4*)(a.q + (int64_t)(mine.start + token) * a.q_stride + (int64_t)head * 128);
    u32x4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = src[F16 && !HAD ? 4 * i + g : 4 * g + i];
    float lse[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = r0 + 4 * quarter + i, of = divided(row < rows ? row : r0, a.per_group);
        lse[i] = a.lse[(int64_t)(mine.start + of) * (a.c.num_heads * a.group) + h * a.group + (row < rows ? row : r0) - of * a.group];
        t.place[i] = row < rows && lse[i] != -__builtin_inff() ? first_place + of : -1;        // (a row that has seen nothing gives nothing)
        t.less[i] = lse[i] * -kLog2e;
    }
    if (HAD) {
        hadamard_row(w, lane);
        if (F16) {                                         // (dimensions 32 g + 8 i to 32 i + 8 g: lanes (n, 0 .. 3) trade pieces)
            u32x4 other[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u32 pick = 0;
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const u32 v = (u32)__shfl((int)w[m][j], 16 * i + n, 64);
                        pick = g == m ? v : pick;
                    }
                    other[i][j] = pick;
                }
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = other[i];
        }
    }
    if (!F16) {
        float all = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const f16x2 p = as_f16x2(w[i >> 2][i & 3]);
            all += (float)p[0] + (float)p[1];
        }
        const float slope = quarters_sum(all) * -(kLog2e * kScale);
#pragma unroll
        for (int i = 0; i < 4; ++i) t.slope[i] = __shfl(slope, 4 * quarter + i, 64);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) t.q[i] = F16 ? w[i] : query_for_numbers(w[i]);
    return t;
}

// ALIGNED: pages of a multiple of 16 positions, so that every 16 positions lie in one page
// ROWS: 4, 8: no more than that many; 16: any number.
template <bool F16, bool ALIGNED, bool HAD, int ROWS>
__global__ __launch_bounds__(64 * kWaves, F16 ? (ROWS == 4 ? 3 : 2) : (ROWS < 16 ? 4 : 3)) void weights_rows_kernel(Weights a, Divisor pages) {
    const PagedKV& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int id = divided(blockIdx.x, a.per_block), first_block = blockIdx.x - id * a.blocks, b = divided(id, a.per_head), h = id - b * c.num_heads;
    const Fresh mine = fresh_of(a, b);
    const int p0 = c.indptr[b], npages = c.indptr[b + 1] - p0;
    const int len = npages > 0 ? (npages - 1) * c.page_size + c.last_page_offset[b] : 0;
    const int rows = mine.count * a.group, first_place = len - mine.all;
    if (rows == 0) return;
    const int64_t page_slots = (int64_t)c.num_layers * 2 * c.num_heads * c.page_size;
    const int64_t head_slots = ((int64_t)c.layer_idx * 2 * c.num_heads + h) * c.page_size;
    constexpr uint32_t VEC = F16 ? 256 : 64;
    constexpr float kUnit = kLog2e * kScale;
    const int highest = first_place + divided(rows - 1, a.per_group);
    const Steps steps = steps_of<6>(a, first_place, highest);              // blocks of 64 positions that some row sees
    const int stride = a.blocks * kWaves;
    float* const sums = a.sums + ((int64_t)b * c.num_heads + h) * a.capacity;

    struct Place {                     // of the lane's position
        int pos, entry, page;
    };
    auto ask = [&](int block) {
        const int at = steps.at(block < steps.all ? block : steps.all - 1) * 64, pos = at + lane, it = divided(pos, pages);
        const int entry = pos - it * c.page_size;
        const bool in = pos < len && it < npages && (u32)entry < (u32)c.page_size;
        const int page = c.indices[p0 + (in ? it : 0)];
        return Place{pos, entry, in ? page : -1};
    };
    struct Block {
        u32x4 k[4][F16 ? 4 : 1];
        u32 param;                     // of the lane's own position
        float before;
    };
    auto there = [&](const Place& p) { return p.page >= 0 && p.page < c.num_pages; };
    auto fetch = [&](Block& f, const Place& p) {           // (a position that is not there reads the first entries of page 0, for nothing)
        const bool is = there(p);
        const int64_t slot = is ? p.page * page_slots + head_slots + p.entry : head_slots;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (ALIGNED) {
                const int page = __builtin_amdgcn_readlane(is ? p.page : -1, 16 * s), entry = __builtin_amdgcn_readlane(p.entry, 16 * s);
                const int64_t base = page >= 0 ? page * page_slots + head_slots + entry : head_slots;
                uint32_t off = (uint32_t)n * VEC + (uint32_t)g * 16;
                asm volatile("" : "+v"(off));                                      // (a 32-bit offset behind wave-uniform addresses)
                const uint8_t* const kd = c.data + base * VEC;
#pragma unroll
                for (int i = 0; i < (F16 ? 4 : 1); ++i) f.k[s][i] = *(const u32x4*)(kd + off + 64 * i);
            } else {
                const int64_t base = __shfl(slot, 16 * s + n, 64);
                const uint8_t* const kd = c.data + base * VEC + g * 16;
#pragma unroll
                for (int i = 0; i < (F16 ? 4 : 1); ++i) f.k[s][i] = *(const u32x4*)(kd + 64 * i);
            }
        }
        f.param = F16 ? 0u : c.param[slot];
        f.before = is && p.pos < a.capacity ? sums[p.pos] : 0.f;
    };
    int block = first_block * kWaves + wave;
    __shared__ u32x4 staged[ROWS == 16 ? 4 : 1][7][64];
    const bool in_lds = ROWS == 16 && rows > 16 && rows <= 64;
    if (in_lds) {
        if (16 * wave < rows) {
            const RowTile<F16> t = row_tile<F16, HAD>(a, mine, h, 16 * wave, rows, first_place, lane, g);
#pragma unroll
            for (int i = 0; i < 4; ++i) staged[wave % (ROWS == 16 ? 4 : 1)][i][lane] = t.q[i];
            staged[wave % (ROWS == 16 ? 4 : 1)][4][lane] = u32x4{as_u32(t.slope[0]), as_u32(t.slope[1]), as_u32(t.slope[2]), as_u32(t.slope[3])};
            staged[wave % (ROWS == 16 ? 4 : 1)][5][lane] = u32x4{as_u32(t.less[0]), as_u32(t.less[1]), as_u32(t.less[2]), as_u32(t.less[3])};
            staged[wave % (ROWS == 16 ? 4 : 1)][6][lane] = u32x4{(u32)t.place[0], (u32)t.place[1], (u32)t.place[2], (u32)t.place[3]};
        }
        __syncthreads();
    }
    auto tile_of = [&](int r0) {
        if (!in_lds) return row_tile<F16, HAD>(a, mine, h, r0, rows, first_place, lane, ROWS == 4 ? 0 : ROWS == 8 ? g & 1 : g);
        RowTile<F16> t;
#pragma unroll
        for (int i = 0; i < 4; ++i) t.q[i] = staged[(r0 >> 4) % (ROWS == 16 ? 4 : 1)][i][lane];
        const u32x4 slope = staged[(r0 >> 4) % (ROWS == 16 ? 4 : 1)][4][lane], less = staged[(r0 >> 4) % (ROWS == 16 ? 4 : 1)][5][lane], place = staged[(r0 >> 4) % (ROWS == 16 ? 4 : 1)][6][lane];
#pragma unroll
        for (int i = 0; i < 4; ++i) t.slope[i] = as_f32(slope[i]), t.less[i] = as_f32(less[i]), t.place[i] = (int)place[i];
        return t;
    };
    if (block >= steps.all) return;
    const CodeMasks masks = code_masks();
    Place here = ask(block), next = ask(block + stride);
    Block f;
    fetch(f, here);
    RowTile<F16> tile = tile_of(0);
    for (;;) {
        const int at = __builtin_amdgcn_readfirstlane(here.pos);
        u32x4 k[4][F16 ? 4 : 1];
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int i = 0; i < (F16 ? 4 : 1); ++i) k[s][i] = f.k[s][i];
        const u32 param = f.param;
        const float before = f.before;
        const Place now = here;
        const bool more = block + stride < steps.all;
        if (more) {
            here = next, next = ask(block + 2 * stride);
            fetch(f, here);
        }
        auto products = [&](f32x4 (&x)[4]) {
#pragma unroll
            for (int s = 0; s < 4; ++s) x[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    u32x4 key;
                    if (F16) {
                        key = k[s][F16 ? i : 0];
                    } else {
                        u32 w = k[s][0][i];
                        asm volatile("" : "+v"(w));        // (unpacked here, tile by tile of rows: all of them are 64 registers)
                        key = numbers_of(w, masks);
                    }
                    x[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, tile.q[i]), __builtin_bit_cast(f16x8, key), x[s], 0, 0, 0);
                }
        };
        // the weights of four rows at the positions p of the lanes, whose keys' parameters are given: added up
        auto weigh = [&](const f32x4& x, u32 key_param, int p, int r0) {
            const f16x2 kp = as_f16x2(key_param);
            const float scale = F16 ? kUnit : (float)kp[0] * kUnit, zero = (float)kp[1];
            const int lowest = first_place + divided(r0, a.per_group), last = first_place + divided((r0 + 15 < rows ? r0 + 16 : rows) - 1, a.per_group);
            const bool all_see = at + 63 <= lowest && (a.window == 0 || at > last - a.window || at + 63 < a.sinks);
            float y[4], sum = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[i] = F16 ? __builtin_fmaf(x[i], scale, tile.less[i]) : __builtin_fmaf(x[i], scale, __builtin_fmaf(zero, tile.slope[i], tile.less[i]));
            if (all_see) {
#pragma unroll
                for (int i = 0; i < 4; ++i) sum += tile.place[i] >= 0 ? __builtin_amdgcn_exp2f(y[i]) : 0.f;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int high = tile.place[i] - at;
                    const bool sees = (p <= high) & ((a.window == 0) | (p > high - a.window) | (p < a.sinks - at));
                    sum += sees ? __builtin_amdgcn_exp2f(y[i]) : 0.f;
                }
            }
            return sum;
        };
        float total = 0.f;
        if constexpr (ROWS < 16) {
            // Register i of lane (n, g) is row 4 g + i: half of the lanes, or three quarters, would have nothing to weigh.  They take the rows of other positions.
            f32x4 x[4];
            products(x);
            auto swapped32 = [](float u, float v) { return as_f32(__builtin_amdgcn_permlane32_swap(as_u32(u), as_u32(v), false, false)[0]); };      // lower halves of both
            auto swapped16 = [](float u, float v) { return as_f32(__builtin_amdgcn_permlane16_swap(as_u32(u), as_u32(v), false, false)[0]); };      // even quarters of both
            f32x4 even, odd;
#pragma unroll
            for (int i = 0; i < 4; ++i) even[i] = swapped32(x[0][i], x[2][i]), odd[i] = swapped32(x[1][i], x[3][i]);
            if (ROWS == 4) {
#pragma unroll
                for (int i = 0; i < 4; ++i) even[i] = swapped16(even[i], odd[i]);              // quarter g: rows 0 .. 3 of its own positions
                total = weigh(even, param, lane, 0);
            } else {
                const int p = 32 * (lane >> 5) + n;        // quarters 0 and 1: positions 0 .., 16 .. (odd); 2 and 3: 32 .., 48 ..
                const u32x2 s0 = both_halves<16>(as_u32(weigh(even, (u32)__shfl((int)param, p, 64), p, 0)));
                const u32x2 s1 = both_halves<16>(as_u32(weigh(odd, (u32)__shfl((int)param, p + 16, 64), p + 16, 0)));
                total = g & 1 ? as_f32(s1.x) + as_f32(s1.y) : as_f32(s0.x) + as_f32(s0.y);
            }
        } else {
            float sum[4] = {0.f, 0.f, 0.f, 0.f}, before_tiles[4] = {0.f, 0.f, 0.f, 0.f};
            u32 params[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) params[s] = F16 ? 0u : (u32)__shfl((int)param, 16 * s + n, 64);
            for (int r0 = 0; r0 < rows; r0 += 16) {
                if (r0 > 0) {
                    tile = tile_of(r0);
                    if ((r0 & 255) == 0) {                 // (sums of 16 tiles, then of these: a long chain of additions would lose what is small)
#pragma unroll
                        for (int s = 0; s < 4; ++s) before_tiles[s] += sum[s], sum[s] = 0.f;
                    }
                }
                f32x4 x[4];
                products(x);
#pragma unroll
                for (int s = 0; s < 4; ++s) sum[s] += weigh(x[s], params[s], 16 * s + n, r0);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const float all = quarters_sum(sum[s] + before_tiles[s]);
                total = g == s ? all : total;
            }
        }
        if (there(now) && now.pos < a.capacity) sums[now.pos] = before + total;
        if (!more) break;
        block += stride;
        if (ROWS == 16 && rows > 16) tile = tile_of(0);
    }
}

// ---- many rows -----------------------------------------------------------------------------------------------------------------------------
// Four waves of 64 positions each, whose keys stay in their registers; the rows come past in units of 32, which the waves share in LDS.  A first launch lays the
// queries out as the matrix instructions take them, so that a unit goes from memory to LDS as it lies, without registers, and is read without
// bank conflicts: eight operands of 1 KB (lane (n, h): dimensions 64 h + 8 i .. of row n) and a ninth, the line: what a logit has besides the codes' product,
// zero sum(q) and the row's logarithm, as a product of bf16 pieces that hold 24 bits together.
// 2048 after 14336, 64 on 8 heads: 522 - 557 us on several cards, 925 - 990 TFLOP/s, with the line's products a ninth more, of a large library product's 1185; 14 of them the
// first launch.  The matrix unit is busy for half of the cycles, the vector unit (a product's exponentials, 32 rows by 64 positions) for the other half, and the clock is down to
// 2.0 GHz.  Slower: three workgroups to a CU with stages half as large (599 against 522), products and exponentials of two units laid between each other (581), a wave's
// products or its exponentials at a higher priority (3 %).
constexpr int kUnitBytes = 9 * 1024, kStageUnits = 4;
constexpr float kNothing = -3e38f;                         // minus the logarithm of a row that gives nothing

__device__ __forceinline__ u32 tops(float lo, float hi) { return __builtin_amdgcn_perm(as_u32(hi), as_u32(lo), 0x07060302u); }
__device__ __forceinline__ float top(float v) { return as_f32(as_u32(v) & 0xFFFF0000u); }
// where the units of a sequence begin: behind those of the sequences before it, whose last units may be filled in part
__device__ __forceinline__ int64_t first_unit(const Weights& a, int start, int b) { return (int64_t)start * a.group / 32 + b; }

template <bool F16>
__global__ __launch_bounds__(256) void weights_queries_kernel(Weights a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hh = lane >> 5;
    const int id = divided(blockIdx.x, a.per_block), first = blockIdx.x - id * a.blocks, b = divided(id, a.per_head), h = id - b * a.c.num_heads;
    const Fresh mine = fresh_of(a, b);
    const int rows = mine.count * a.group;
    for (int unit = first * 4 + wave; unit * 32 < rows; unit += a.blocks * 4) {
        const int row = unit * 32 + n, r = row < rows ? row : rows - 1;        // (the last unit is filled up with the last row, which gives nothing there)
        const int t = divided(r, a.per_group), head = h * a.group + r - t * a.group;
        const u32x4* const src = (const u32x4*)(a.q + (int64_t)(mine.start + t) * a.q_stride + (int64_t)head * 128) + 8 * hh;
        const float lse = a.lse[(int64_t)(mine.start + t) * (a.c.num_heads * a.group) + head];
        u32x4 w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = src[i];
        if (a.q_had) {
            float v[64];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const f16x2 p = as_f16x2(w[i >> 2][i & 3]);
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
                const u32x2 e = both_halves<32>(as_u32(v[i]));
                v[i] = hh ? as_f32(e.x) - as_f32(e.y) : as_f32(e.x) + as_f32(e.y);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) w[i >> 2][i & 3] = narrow_f16x2(v[2 * i] * kScale, v[2 * i + 1] * kScale);
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const f16x2 p = as_f16x2(w[i >> 2][i & 3]);
            sum += (float)p[0] + (float)p[1];
        }
        const u32x2 both = both_halves<32>(as_u32(sum));
        const float all = as_f32(both.x) + as_f32(both.y);
        float m = lse * -kLog2e;
        m = row >= rows || __builtin_fabsf(m) > 3e38f ? kNothing : m != m ? __builtin_nanf("") : m;
        // (a row that gives nothing may hold anything; its infinities and NaN would get into the sums)
        const bool nothing = m == kNothing && !(__builtin_fabsf(all) < 3e38f);
        const float s = nothing ? 0.f : all * -(kLog2e * kScale), s1 = top(s), s2 = top(s - s1), s3 = s - s1 - s2;
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = nothing ? u32x4{0, 0, 0, 0} : w[i];
        const float m1 = top(m), m2 = top(m - m1), m3 = m - m1 - m2;
        uint8_t* const to = a.units + ((int64_t)h * a.all_units + first_unit(a, mine.start, b) + unit) * kUnitBytes + lane * 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) *(u32x4*)(to + 1024 * i) = F16 ? w[i] : query_for_numbers(w[i]);
        *(u32x4*)(to + 8192) = hh ? u32x4{tops(m3, 0.f), 0, 0, 0} : u32x4{tops(s1, s2), tops(s3, s1), tops(s2, s3), tops(m1, m2)};
    }
}

typedef __attribute__((address_space(1))) const void* GlobalPtr;
typedef __attribute__((address_space(3))) void* LdsPtr;

template <bool F16>
__global__ __launch_bounds__(256, 2) void weights_tiles_kernel(Weights a, Divisor pages) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][kStageUnits * kUnitBytes];
    const PagedKV& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, hh = lane >> 5;
    // (a head's workgroups are on one XCD where 8 divides the heads; blocks that most rows see come first)
    const int items = c.batch_size * c.num_heads;
    const int turn = blockIdx.x / items, id = blockIdx.x - turn * items, b = divided(id, a.per_head), h = id - b * c.num_heads;
    const int first_block = turn / a.splits, split = turn - first_block * a.splits;
    const Fresh mine = fresh_of(a, b);
    const int p0 = c.indptr[b], npages = c.indptr[b + 1] - p0;
    const int len = npages > 0 ? (npages - 1) * c.page_size + c.last_page_offset[b] : 0;
    const int rows = mine.count * a.group, first_place = len - mine.all;
    if (rows == 0) return;
    const int64_t page_slots = (int64_t)c.num_layers * 2 * c.num_heads * c.page_size;
    const int64_t head_slots = ((int64_t)c.layer_idx * 2 * c.num_heads + h) * c.page_size;
    constexpr uint32_t VEC = F16 ? 256 : 64;
    constexpr float kUnit = kLog2e * kScale;
    const int highest = first_place + divided(rows - 1, a.per_group);
    const Steps steps = steps_of<8>(a, first_place, highest);              // blocks of 256 positions that some row sees
    const uint8_t* const units = a.units + ((int64_t)h * a.all_units + first_unit(a, mine.start, b)) * kUnitBytes;
    // Row r is of token r / group, so it sees the position `pos` if it is not before `seen_from` and before `seen_to`
    auto seen_from = [&](int pos) {
        const int t = pos - first_place;                   // the token at that position
        return t <= 0 ? 0 : t >= mine.count ? rows : t * a.group;
    };
    auto seen_to = [&](int pos) {
        if (a.window == 0 || pos < a.sinks) return rows + 32;              // (rows that only fill up give nothing by themselves)
        const int64_t t = (int64_t)pos + a.window - first_place;
        return t <= 0 ? 0 : t >= mine.count ? rows + 32 : (int)t * a.group;
    };

    for (int block = first_block; block < steps.all; block += a.blocks) {
        const bool whole = a.splits == 1 || block >= a.blocks;             // (blocks that the launch was not sized for are not split)
        if (whole && split > 0) break;
        const int block_at = steps.at(block) * 256, at = block_at + 64 * wave;
        const int pos = at + lane, it = divided(pos, pages);
        const u32 entry = (u32)(pos - it * c.page_size);
        const bool in = pos < len && it < npages && entry < (u32)c.page_size;
        const int page = c.indices[p0 + (in ? it : 0)];
        const bool there = in && page >= 0 && page < c.num_pages;
        const int64_t slot = there ? page * page_slots + head_slots + entry : head_slots;
        const u32 param = F16 ? 0u : c.param[slot];
        const CodeMasks masks = code_masks();
        u32x4 k[2][8], line[2];
        float slope[2];
        int from[2], to[2];
#pragma unroll
        for (int cb = 0; cb < 2; ++cb) {
            const uint8_t* const kd = c.data + __shfl(slot, 32 * cb + n, 64) * VEC + hh * (VEC / 2);
            if (F16) {
#pragma unroll
                for (int i = 0; i < 8; ++i) k[cb][i] = *(const u32x4*)(kd + 16 * i);
            } else {
                const u32x4 w0 = *(const u32x4*)kd, w1 = *(const u32x4*)(kd + 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) k[cb][i] = numbers_of(w0[i], masks), k[cb][4 + i] = numbers_of(w1[i], masks);
            }
            const f16x2 p = as_f16x2((u32)__shfl((int)param, 32 * cb + n, 64));
            slope[cb] = F16 ? kUnit : (float)p[0] * kUnit;
            const float zero = F16 ? 0.f : (float)p[1], z1 = top(zero), z2 = zero - z1;
            line[cb] = hh ? u32x4{0x00003F80u, 0, 0, 0} : u32x4{tops(z1, z1), tops(z1, z2), tops(z2, z2), 0x3F803F80u};
            from[cb] = seen_from(at + 32 * cb + n), to[cb] = seen_to(at + 32 * cb + n);
        }
        // rows that see one of the workgroup's positions; those that see all of the wave's, and those that see any
        const int last_seen = a.window == 0 || block_at < a.sinks ? rows : seen_to(block_at + 255);
        int u_begin = seen_from(block_at) / 32, u_end = ((last_seen < rows ? last_seen : rows) + 31) / 32;
        if (!whole) {
            const int all = u_end > u_begin ? u_end - u_begin : 0, first = u_begin;
            u_begin = first + (int)((int64_t)all * split / a.splits), u_end = first + (int)((int64_t)all * (split + 1) / a.splits);
        }
        const int all_from = seen_from(at + 63), all_to = at + 63 < a.sinks ? rows + 32 : seen_to(at < a.sinks ? a.sinks : at);
        const int any_from = seen_from(at), any_to = a.window == 0 || at < a.sinks ? rows + 32 : seen_to(at + 63);

        auto fetch = [&](int stage, int buffer) {          // units u_begin + 4 stage .. into LDS; each wave takes a fourth of their pieces of 1 KB
            const int u = u_begin + stage * kStageUnits;
#pragma unroll
            for (int i = 0; i < 9; ++i) {
                const int piece = 4 * i + wave;
                if (u + piece / 9 < u_end)
                    __builtin_amdgcn_global_load_lds((GlobalPtr)(units + (int64_t)u * kUnitBytes + piece * 1024 + lane * 16), (LdsPtr)(&lds[buffer][piece * 1024]), 16, 0, 0);
            }
        };
        float sum[2] = {0.f, 0.f}, total[2] = {0.f, 0.f}, lost[2] = {0.f, 0.f};
        const int stages = (u_end - u_begin + kStageUnits - 1) / kStageUnits;
        if (stages > 0) fetch(0, 0);
        for (int stage = 0; stage < stages; ++stage) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();                               // this stage is in LDS, and nobody reads the last one's any more
            if (stage + 1 < stages) fetch(stage + 1, stage + 1 & 1);
            const uint8_t* const buffer = lds[stage & 1];
#pragma unroll 1
            for (int i = 0; i < kStageUnits; ++i) {
                const int u = u_begin + stage * kStageUnits + i, r0 = u * 32;
                if (u >= u_end || r0 + 31 < any_from || r0 >= any_to) continue;
                const uint8_t* const from_lds = buffer + i * kUnitBytes + lane * 16;
                f32x16 x[2], t[2];
                const u32x4 q_line = *(const u32x4*)(from_lds + 8192);
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[cb][j] = t[cb][j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const f16x8 q = *(const f16x8*)(from_lds + 1024 * j);
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb) x[cb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(q, __builtin_bit_cast(f16x8, k[cb][j]), x[cb], 0, 0, 0);
                }
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) t[cb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, q_line), __builtin_bit_cast(bf16x8, line[cb]), t[cb], 0, 0, 0);
                if (r0 >= all_from && r0 + 32 <= all_to) {
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb) {
                        float s0 = 0.f, s1 = 0.f;
#pragma unroll
                        for (int j = 0; j < 16; j += 2) {
                            s0 += __builtin_amdgcn_exp2f(__builtin_fmaf(x[cb][j], slope[cb], t[cb][j]));
                            s1 += __builtin_amdgcn_exp2f(__builtin_fmaf(x[cb][j + 1], slope[cb], t[cb][j + 1]));
                        }
                        sum[cb] += s0 + s1;
                    }
                } else {
#pragma unroll
                    for (int cb = 0; cb < 2; ++cb) {
                        float s0 = 0.f;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const int r = r0 + 8 * (j >> 2) + 4 * hh + (j & 3);
                            const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(x[cb][j], slope[cb], t[cb][j]));
                            s0 += r >= from[cb] && r < to[cb] ? e : 0.f;
                        }
                        sum[cb] += s0;
                    }
                }
            }
            if ((stage & 3) == 3 || stage + 1 == stages) {
                // (what is lost of a small sum added to a large one is kept for the next)
#pragma unroll
                for (int cb = 0; cb < 2; ++cb) {
                    const float more = sum[cb] - lost[cb], now = total[cb] + more;
                    lost[cb] = (now - total[cb]) - more, total[cb] = now, sum[cb] = 0.f;
                }
            }
        }
        float all[2];
#pragma unroll
        for (int cb = 0; cb < 2; ++cb) {
            const u32x2 both = both_halves<32>(as_u32(total[cb]));
            all[cb] = as_f32(both.x) + as_f32(both.y);
        }
        if (!whole) a.part[(((int64_t)split * items + id) * a.blocks + block) * 256 + 64 * wave + lane] = there ? (hh ? all[1] : all[0]) : 0.f;
        else if (there && pos < a.capacity) a.sums[((int64_t)b * c.num_heads + h) * a.capacity + pos] += hh ? all[1] : all[0];
        __syncthreads();                                   // (the next block's first stage overwrites LDS)
    }
}

// The sums of the rows' splits -> the positions' sums, in the splits' order
__global__ __launch_bounds__(256) void weights_join_kernel(Weights a) {
    const PagedKV& c = a.c;
    const int items = c.batch_size * c.num_heads, block = blockIdx.x / items, id = blockIdx.x - block * items, b = divided(id, a.per_head);
    const Fresh mine = fresh_of(a, b);
    const int npages = c.indptr[b + 1] - c.indptr[b], len = npages > 0 ? (npages - 1) * c.page_size + c.last_page_offset[b] : 0;
    const int rows = mine.count * a.group, first_place = len - mine.all;
    if (rows == 0) return;
    const Steps steps = steps_of<8>(a, first_place, first_place + divided(rows - 1, a.per_group));
    const int pos = steps.at(block) * 256 + (int)threadIdx.x;
    if (block >= steps.all || pos >= len || pos >= a.capacity) return;
    const float* const src = a.part + ((int64_t)id * a.blocks + block) * 256 + threadIdx.x;
    float sum = 0.f;
    for (int s = 0; s < a.splits; ++s) sum += src[(int64_t)s * items * a.blocks * 256];
    a.sums[(int64_t)id * a.capacity + pos] += sum;
}

// Which kernel, workgroups per (sequence, key head), and among how many of them the rows are split
struct WeightsPlan {
    bool tiles;
    int splits;
    int64_t blocks, most;              // most: workgroups of a launch, which has fewer than 2^32 threads
};
WeightsPlan weights_plan(bool fp16, int64_t rows, int64_t tokens, int group, int64_t num_heads, int64_t batch, int64_t max_new_len, int64_t seen) {
    if (max_new_len <= 0 || max_new_len > tokens) max_new_len = tokens;
    WeightsPlan p;
    p.tiles = max_new_len * group > 64;
    p.splits = 1;
    p.most = 0xffffffffll / 256;
    p.blocks = (seen + 255) / 256;
    const int64_t cus = qr_device().cus, items = batch * num_heads;
    if (!p.tiles) {                    // workgroups that are on the chip at once, of equal work
        const int64_t room = (fp16 ? (rows <= 4 ? 3 : 2) : (rows <= 8 ? 4 : 3)) * cus / items, all = (seen + 63) / 64;
        const int64_t turns = room > 0 ? (all + 4 * room - 1) / (4 * room) : all;
        if (turns > 1) p.blocks = (all + 4 * turns - 1) / (4 * turns);
    }
    if (p.blocks > 0xffff) p.blocks = 0xffff;
    if (items * p.blocks > p.most) p.blocks = items < p.most ? p.most / items : 1;
    if (p.tiles) {
        // Parts of the rows: microseconds of a workgroup's unit of 32 rows, alone on its CU 0.74, with another one 0.98, what goes around its units 6, the join 4 and
        // 0.0003 for a part of a block.  (8192 rows of one key head, one block: 193 us whole, 112, 72, 48, 32 and 27 in 2, 4, 8, 16 and 32 parts; 536 blocks of
        // 8192 rows, two rounds of which the second is nearly empty: 403 whole, 328 in four parts; 512 rows of a block 24.5, in eight parts 13.7.)
        const int64_t units = (max_new_len * group + 31) / 32, all = items * p.blocks;
        float least = -1.f;
        for (int splits = 1; splits <= 32 && (splits == 1 || (2 * splits <= units && all * splits <= p.most)); ++splits) {
            const float each = all * splits <= cus ? 0.74f : 0.98f;
            const float time = (float)((all * splits + 2 * cus - 1) / (2 * cus)) * ((float)((units + splits - 1) / splits) * each + 6.f) +
                               (splits > 1 ? 4.f + 0.0003f * (float)(all * splits) : 0.f);
            // (parts for a tenth at least: blocks that few rows see fill rounds up by themselves)
            if (least < 0.f || time < (p.splits == 1 ? 0.9f : 1.f) * least) least = time, p.splits = splits;
        }
    }
    return p;
}
int bounded_window(int64_t window) { return (int)(window > 0x3fffffff ? 0 : window); }       // (longer than any sequence)
int bounded_sinks(int64_t sinks) { return (int)(sinks > 0x3fffffff ? 0x3fffffff : sinks); }
int64_t weights_units(int64_t tokens, int group, int64_t batch) { return tokens * group / 32 + batch + 2; }
// workspace: the queries' units, then the splits' sums
size_t weights_bytes(const WeightsPlan& p, int64_t tokens, int group, int64_t num_heads, int64_t batch) {
    if (!p.tiles) return 0;
    return (size_t)weights_units(tokens, group, batch) * num_heads * kUnitBytes + (p.splits > 1 ? (size_t)p.splits * batch * num_heads * p.blocks * 1024 : 0);
}
// positions that the launch is sized for (what is longer is gone through in turns)
int64_t seen_positions(int64_t tokens, int64_t max_new_len, int64_t max_seq_len, int64_t window, int64_t sinks, int64_t capacity) {
    int64_t seen = max_seq_len > 0 && max_seq_len < capacity ? max_seq_len : capacity;
    const int64_t fresh = max_new_len > 0 && max_new_len < tokens ? max_new_len : tokens;
    if (window > 0 && window < seen && sinks < seen && seen > window + fresh + sinks + 768) seen = window + fresh + sinks + 768;
    return seen;
}

using Kernel = void (*)(Weights, Divisor);
template <bool F16, int ROWS>
Kernel rows_kernel(bool aligned, bool had) {
    return had ? (aligned ? weights_rows_kernel<F16, true, true, ROWS> : weights_rows_kernel<F16, false, true, ROWS>)
               : (aligned ? weights_rows_kernel<F16, true, false, ROWS> : weights_rows_kernel<F16, false, false, ROWS>);
}

template <bool F16>
int launch_weights(const WeightsPlan& plan, Weights a, hipStream_t st) {
    const int64_t items = (int64_t)a.c.batch_size * a.c.num_heads;
    const Divisor pages = divisor_of(a.c.page_size);
    if (plan.tiles) {
        // (a wave of the first launch takes the units of a (sequence, key head) in turns)
        int64_t each = ((int64_t)a.tokens * a.group / 32 / a.c.batch_size + 4) / 4, most = plan.most / items;
        each = each > most ? most : each;
        Weights first = a;
        first.blocks = (int)each, first.per_block = divisor_of(each);
        weights_queries_kernel<F16><<<dim3((unsigned)(items * each)), dim3(256), 0, st>>>(first);
        weights_tiles_kernel<F16><<<dim3((unsigned)(items * a.blocks * a.splits)), dim3(256), 0, st>>>(a, pages);
        if (a.splits > 1) weights_join_kernel<<<dim3((unsigned)(items * a.blocks)), dim3(256), 0, st>>>(a);
    } else {
        const bool aligned = a.c.page_size % 16 == 0;
        const Kernel kernel = a.rows <= 4 ? rows_kernel<F16, 4>(aligned, a.q_had) : a.rows <= 8 ? rows_kernel<F16, 8>(aligned, a.q_had) : rows_kernel<F16, 16>(aligned, a.q_had);
        kernel<<<dim3((unsigned)(items * a.blocks)), dim3(64 * kWaves), 0, st>>>(a, pages);
    }
    return qr_launch_status();
}

int accumulate(bool fp16, void* weights, int64_t capacity, const void* q, int64_t q_stride, int q_had_mode, const void* lse, const void* starts, int64_t tokens,
               int num_q_heads, const void* kv_data, const void* kv_param, const void* kv_indptr, const void* kv_indices, const void* last_page_offset, int64_t num_pages,
               int num_layers, int layer_idx, int num_heads, int page_size, int head_dim, int64_t batch_size, int64_t max_new_len, int64_t max_seq_len, int64_t window,
               int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = qr_internal_check_paged_cache(kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads, page_size,
                                                 head_dim, batch_size);
    if (rc != QR_OK) return rc;
    if (q_had_mode != 0 && q_had_mode != 1) return QR_E_DTYPE;
    if (tokens < 0 || num_q_heads <= 0 || num_q_heads % num_heads || window < 0 || sinks < 0 || max_new_len < 0 || max_seq_len < 0 || capacity < 0) return QR_E_SHAPE;
    if (tokens == 0 || batch_size == 0 || capacity == 0) return QR_OK;
    if (!starts && tokens != batch_size) return QR_E_SHAPE;
    if (!weights || !q || !lse) return QR_E_NULL;
    if (((uintptr_t)q & 15) || ((uintptr_t)weights & 3) || ((uintptr_t)lse & 3) || q_stride % 8) return QR_E_ALIGN;
    if (q_stride < (int64_t)num_q_heads * 128 || tokens > 0x3fffffff || tokens * num_q_heads > 0x3fffffff || num_q_heads / num_heads > 1024 || num_heads > 65536)
        return QR_E_SHAPE;
    Weights a;
    a.c = qr_internal_paged_kv((void*)kv_data, (void*)kv_param, kv_indptr, kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads, page_size, batch_size);
    a.q = (const f16*)q, a.lse = (const float*)lse, a.sums = (float*)weights;
    a.starts = (const int32_t*)starts;
    a.q_stride = q_stride, a.capacity = capacity;
    a.tokens = (int)tokens, a.group = num_q_heads / num_heads;
    a.window = bounded_window(window), a.sinks = bounded_sinks(sinks);
    a.q_had = q_had_mode;
    a.rows = starts ? tokens * a.group : a.group;          // (by bounds, which are on the device, one sequence may have all of them)
    a.per_group = divisor_of(a.group), a.per_head = divisor_of(num_heads);
    const int64_t fresh = starts ? max_new_len : 1;
    WeightsPlan plan = weights_plan(fp16, a.rows, tokens, a.group, num_heads, batch_size, fresh, seen_positions(tokens, fresh, max_seq_len, a.window, a.sinks, capacity));
    a.all_units = weights_units(tokens, a.group, batch_size);
    if (plan.tiles && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < weights_bytes(plan, tokens, a.group, num_heads, batch_size))) plan.tiles = false, plan.splits = 1;
    a.units = (uint8_t*)workspace;
    a.part = (float*)((uint8_t*)workspace + (size_t)a.all_units * num_heads * kUnitBytes);
    a.splits = plan.splits;
    a.blocks = (int)plan.blocks, a.per_block = divisor_of(plan.blocks);
    const int64_t wide = num_heads * plan.blocks * plan.splits, at_once = batch_size * wide <= plan.most ? batch_size : plan.most / wide;
    int lrc = QR_OK;
    for (int64_t first = 0; first < batch_size && lrc == QR_OK; first += at_once) {
        Weights some = a;
        some.c.batch_size = (int)(batch_size - first < at_once ? batch_size - first : at_once);
        some.c.indptr += first, some.c.last_page_offset += first;
        some.sums += first * num_heads * capacity;
        if (a.starts) some.starts += first;
        else some.q += first * q_stride, some.lse += first * num_q_heads;
        lrc = fp16 ? launch_weights<true>(plan, some, (hipStream_t)stream) : launch_weights<false>(plan, some, (hipStream_t)stream);
    }
    return lrc;
}

}  // namespace

extern "C" size_t qr_accumulate_weights_workspace_bytes(int fp16_pages, int64_t capacity, int64_t tokens, int num_q_heads, int num_heads, int64_t batch_size,
                                                        int64_t max_new_len, int64_t max_seq_len, int64_t window, int64_t sinks) {
    if (tokens <= 0 || num_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_heads || batch_size <= 0 || batch_size > 0x7fffffff || tokens > 0x3fffffff ||
        tokens * num_q_heads > 0x3fffffff || num_q_heads / num_heads > 1024 || num_heads > 65536 || capacity <= 0)
        return 0;                                          // (the call itself refuses them, or has nothing to do)
    const int group = num_q_heads / num_heads;
    return weights_bytes(weights_plan(fp16_pages != 0, tokens * group, tokens, group, num_heads, batch_size, max_new_len,
                                      seen_positions(tokens, max_new_len, max_seq_len, bounded_window(window), bounded_sinks(sinks), capacity)),
                         tokens, group, num_heads, batch_size);
}

#define QR_WEIGHTS_ENTRY(NAME, FP16)                                                                                                                     \
    extern "C" int NAME(void* weights, int64_t capacity, const void* q, int64_t q_stride, int q_had_mode, const void* lse,                               \
                        const void* seqlen_indptr_or_null, int64_t tokens, int num_q_heads, const void* kv_data, const void* kv_param,                   \
                        const void* kv_indptr, const void* kv_indices, const void* last_page_offset, int64_t num_pages, int num_layers, int layer_idx,   \
                        int num_heads, int page_size, int head_dim, int64_t batch_size, int64_t max_new_len, int64_t max_seq_len, int64_t window,        \
                        int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {                                                                                                   \
        return accumulate(FP16, weights, capacity, q, q_stride, q_had_mode, lse, seqlen_indptr_or_null, tokens, num_q_heads, kv_data, kv_param, kv_indptr, \
                          kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads, page_size, head_dim, batch_size, max_new_len,       \
                          max_seq_len, window, sinks, workspace, workspace_bytes, stream);                                                                                           \
    }
QR_WEIGHTS_ENTRY(qr_accumulate_weights_i4, false)
QR_WEIGHTS_ENTRY(qr_accumulate_weights_f16, true)
