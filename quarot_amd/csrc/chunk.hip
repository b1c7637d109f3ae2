// Attention of new tokens over the paged KV cache: every sequence brings any number of them, each sees the cached positions up to its own
// (all of them, or the last `window` and the first `sinks`), and several query heads may share a key head.
//
//   o[t, h] = sum_j softmax_j( q[t, h] . k[j, h / G] / sqrt(128) ) v[j, h / G]      over j <= P(t) and (P(t) - j < window or j < sinks)
//
// with P(t) = (tokens the sequence holds) - (its new tokens) + (which of them t is).  A row that sees no position is zero.
//
// Int4 pages hold x = code * scale - zero.  Both products run on the codes themselves, which fp16 holds exactly, so that no cached value is
// rounded:
//   q . k_j = scale_j (q . code_j) - zero_j sum(q)                                 (the last factor once per row)
//   sum_j p_j v_j = sum_j (p_j f_j) (2^e_j code_j) - sum_j p_j zero_j              with scale_j = f_j 2^e_j
// Only p_j f_j is rounded to fp16, the matrix instruction's type; f_j lies in [1, 2), so weights of large and of tiny scales have the same range.
// The rounded number over f_j is the weight in every sum, so a rounding (2^-11 at most) changes a weight and nothing else.  Maxima, sums and
// outputs are held in 32 bits.
#include <type_traits>

#include "qr_chunk.h"

namespace {

// ---- few rows ------------------------------------------------------------------------------------------------------------------------------
// A workgroup of NW waves takes 16 NB rows of a (sequence, key head); its waves (and those of the other splits) take the steps of 32
// positions in turn, so a cached vector is read once per tile of rows.  A wave works on transposed tiles, positions x rows: the first product's
// result has a row in every lane and positions in its registers, which is what the second product takes as its right operand, with no exchange
// between lanes.  The contraction's order is free, so a position's codes are used as they lie: lane (n, g) of the first product takes bytes 16 g ..
// of key n, the word s of them in step s (fp16 pages: bytes 64 s + 16 g ..); lane (m, g) of the second takes word m of the eight keys
// 4 g .. 4 g + 3 and 16 + 4 g .. of a step, whose nibble b is row m of its block b of outputs.  A wave has the next step's keys and values under
// way (32 sequences of 4001 in a window, 64 on 8 heads: 20 us, 3.6 TB/s, bound by the vector unit; fp16 pages, 16 x 2500 in a window: 69 us, 4.85 TB/s).
template <bool F16>
struct Fetched {                       // a step's keys, refilled behind the first product, and its values, refilled behind the second
    u32x4 k[F16 ? 8 : 2], kp[F16 ? 1 : 2], vp[F16 ? 1 : 2];
    u32x4 v4[F16 ? 8 : 1];
    u32 v[F16 ? 1 : 8];
};
struct There {
    u32 ok;                            // bit 4 kb + i: position 16 kb + 4 g + i is there
    bool all;                          // all of them are, in every lane
};

// SHARED: a Chunk, else ChunkRows alone (what a Chunk's rows need before the first load and behind the last step is 0.45 of the 7.4 us of a launch of a few steps, its arguments alone
// 0.15).
template <bool SHARED>
using Launch = std::conditional_t<SHARED, Chunk, ChunkRows>;
// ALIGNED: pages of a multiple of 16 positions, so that each half of a step lies in one page.
template <int NB, int NW, bool F16, bool ALIGNED, bool SHARED>
__device__ __forceinline__ void attend_rows(const Launch<SHARED>& a, const Divisor& pages, const int group_number) {
    extern __shared__ __attribute__((aligned(16))) f32x4 st4[];            // per wave and row: maximum, sum, -, -, 128 outputs
    const PagedKV& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int id = divided(group_number, a.per_split), split = group_number - id * a.splits, item = divided(id, a.per_head), h = id - item * c.num_heads;
    int b, first_tile;
    if (!item_of<16 * NB>(a, item, b, first_tile)) return;
    const Fresh mine_tokens = fresh_of(a, b);
    const int start = mine_tokens.start;
    const int p0 = c.indptr[b], npages = c.indptr[b + 1] - p0;
    const int len = npages > 0 ? (npages - 1) * c.page_size + c.last_page_offset[b] : 0;
    const int rows = mine_tokens.count * a.group, first_place = len - mine_tokens.all;        // (the first new token's position)
    const int64_t page_slots = (int64_t)c.num_layers * 2 * c.num_heads * c.page_size;
    const int64_t head_slots = ((int64_t)c.layer_idx * 2 * c.num_heads + h) * c.page_size;
    const int64_t kv_slots = (int64_t)c.num_heads * c.page_size;
    constexpr uint32_t VEC = F16 ? 256 : 64;               // bytes of a vector
    Divisor per_place = a.per_group;
    if constexpr (SHARED) per_place = a.per_place;

    for (int tile = first_tile; tile * 16 * NB < rows; tile += a.tiles) {
        const int r0 = tile * 16 * NB, r1 = r0 + 16 * NB < rows ? r0 + 16 * NB : rows;
        const int lowest = first_place + divided(r0, per_place), highest = first_place + divided(r1 - 1, per_place);
        const Steps steps = steps_of<5>(a, lowest, highest);
        const int stride = NW * a.splits;

        // Loads are unconditional: a position that is not there reads the first entries of page 0 and is masked.  ALIGNED: the page numbers of the wave's next 32
        // steps are held by its lanes, two a step (-1: none), and taken by number: a load of its own per step would be waited for, and with it all that is under way.
        Fetched<F16> f;
        int held_pages = -1, turn = 0;                     // turn: which of the 32 the step is that is fetched next
        int64_t slots[ALIGNED ? 2 : 8];                    // ALIGNED: of the step's halves; else of the lane's eight positions
        auto fetch_pages = [&](int s) {
            const int later = s + (lane >> 1) * stride, it = divided(steps.at(later < steps.all ? later : steps.all - 1) * 32 + 16 * (lane & 1), pages);
            const int page = npages > 0 ? c.indices[p0 + (it < npages ? it : 0)] : -1;
            held_pages = it < npages && page < c.num_pages ? page : -1;
            turn = 0;
        };
        auto fetch_keys = [&](int s) {
            const int at = steps.at(s) * 32;
            There t{0, true};
            if (ALIGNED) {
                uint32_t k_off = (uint32_t)n * VEC + (uint32_t)g * 16, p_off = (uint32_t)g * 16;
                asm volatile("" : "+v"(k_off), "+v"(p_off));                       // (kept as 32-bit offsets behind wave-uniform addresses)
                t.all = at + 32 <= len;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const int pos = at + 16 * kb, page = __builtin_amdgcn_readlane(held_pages, 2 * turn + kb);
                    const u32 entry = (u32)(pos - divided(pos, pages) * c.page_size);
                    const bool there = page >= 0 && entry < (u32)c.page_size;
                    slots[kb] = there ? page * page_slots + head_slots + entry : head_slots;
                    const uint8_t* const kd = c.data + slots[kb] * VEC;
                    if (!there) t.all = false;
                    else t.ok |= 15u << (4 * kb);
#pragma unroll
                    for (int i = 0; i < (F16 ? 4 : 1); ++i) f.k[F16 ? 4 * kb + i : kb] = *(const u32x4*)(kd + k_off + 64 * i);
                    if (!F16) {
                        const uint8_t* const kp = (const uint8_t*)(c.param + slots[kb]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) f.kp[kb][i] = *(const u32*)(kp + p_off + 4 * i);
                    }
                }
                if (!t.all) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (at + 16 * (k >> 2) + 4 * g + (k & 3) >= len) t.ok &= ~(1u << k);
                }
            } else {
                const int pos = at + (lane & 31), it = divided(pos, pages);
                const u32 entry = (u32)(pos - it * c.page_size);
                const bool in = pos < len && it < npages && entry < (u32)c.page_size;
                const int page = npages > 0 ? c.indices[p0 + (in ? it : 0)] : -1;
                const bool mine_ok = in && page >= 0 && page < c.num_pages;
                const int64_t mine = mine_ok ? page * page_slots + head_slots + entry : head_slots;
                t.all = __builtin_amdgcn_ballot_w64(!mine_ok) == 0;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const uint8_t* const kd = c.data + __shfl(mine, 16 * kb + n, 64) * VEC + g * 16;
#pragma unroll
                    for (int i = 0; i < (F16 ? 4 : 1); ++i) f.k[F16 ? 4 * kb + i : kb] = *(const u32x4*)(kd + 64 * i);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        slots[(4 * kb + i) % (ALIGNED ? 2 : 8)] = __shfl(mine, 16 * kb + 4 * g + i, 64);
                        t.ok |= (u32)__shfl((int)mine_ok, 16 * kb + 4 * g + i, 64) << (4 * kb + i);
                        if (!F16) f.kp[kb][i] = c.param[slots[(4 * kb + i) % (ALIGNED ? 2 : 8)]];
                    }
                }
            }
            return t;
        };
        auto fetch_values = [&]() {                        // of the step whose keys were fetched last
            uint32_t v_off = (uint32_t)g * 4 * VEC + (uint32_t)n * (VEC / 16), p_off = (uint32_t)g * 16;
            asm volatile("" : "+v"(v_off), "+v"(p_off));
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t slot = (ALIGNED ? slots[k >> 2] : slots[k % (ALIGNED ? 2 : 8)]) + kv_slots;
                const uint8_t* const vd = c.data + slot * VEC + (ALIGNED ? v_off + VEC * (k & 3) : (uint32_t)n * (VEC / 16));
                if (F16) {
                    f.v4[k] = *(const u32x4*)vd;
                } else {
                    f.v[k] = *(const u32*)vd;
                    f.vp[k >> 2][k & 3] = ALIGNED ? *(const u32*)((const uint8_t*)(c.param + slot) + p_off + 4 * (k & 3)) : c.param[slot];
                }
            }
        };
        int s = split * NW + wave;
        There there{0, false};
        if (s < steps.all) {
            if (ALIGNED) fetch_pages(s);
            there = fetch_keys(s);
            fetch_values();
        }
        __builtin_amdgcn_sched_barrier(0);

        // the queries: lane (n, g) holds dimensions 32 g + 8 i .. + 7 (fp16 pages: 32 i + 8 g ..), i = 0 .. 3, of row n of every block
        u32x4 qf[NB][4];
        float qsum[NB];                                    // minus the row's sum, in units of the products'
        constexpr float kUnit = kLog2e * kScale * (F16 ? 1.f : kCodeUnit);         // of a logit, base 2
        int place[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int r = r0 + 16 * nb + n;
            const bool in = r < rows;
            const int t = divided(in ? r : r0, a.per_group), head = h * a.group + (in ? r : r0) - t * a.group;
            place[nb] = in ? first_place + divided(r, per_place) : -1;
            const u32x4* src = (const u32x4*)(a.q + (int64_t)(start + t) * a.q_stride + (int64_t)head * 128) + (F16 ? g : 4 * g);
            u32x4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = in ? src[F16 ? 4 * i : i] : u32x4{0, 0, 0, 0};
            if (__builtin_expect(a.q_had, 0)) {
                // the Hadamard transform over the head dimension in 32 bits: five of the index's bits within the lane, two across the quarters; rounded to
                // fp16 like the transform's own entry point
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
                    float v = (lane & 16) ? as_f32(e.x) - as_f32(e.y) : as_f32(e.x) + as_f32(e.y);
                    e = both_halves<32>(as_u32(v));
                    t32[i] = (lane & 32) ? as_f32(e.x) - as_f32(e.y) : as_f32(e.x) + as_f32(e.y);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i >> 2][i & 3] = narrow_f16x2(t32[2 * i] * kScale, t32[2 * i + 1] * kScale);
            }
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const f16x2 p = as_f16x2(w[i >> 2][i & 3]);
                sum += (float)p[0] + (float)p[1];
            }
            qsum[nb] = quarters_sum(sum) * (-1.f / kCodeUnit);
#pragma unroll
            for (int i = 0; i < 4; ++i) qf[nb][i] = F16 ? w[i] : query_for_codes(w[i]);
        }

        const CodeMasks masks = code_masks();
        float m[NB], d[NB], pz[NB];
        f32x4 acc[NB][8];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb] = kEmpty, d[nb] = 0.f, pz[nb] = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[nb][k] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

        auto consume = [&](int step, int next) {
            const int at = steps.at(step) * 32;
            const There ok = there;
            const bool whole = ok.all && at + 31 <= lowest && (a.window == 0 || at > highest - a.window || at + 31 < a.sinks);
            auto sees = [&](int nb, int k) {               // whether the lane's row sees its position k
                const int pos = at + 16 * (k >> 2) + 4 * g + (k & 3);
                return pos <= place[nb] && (a.window == 0 || pos > place[nb] - a.window || pos < a.sinks) && (ok.ok >> k & 1);
            };
            // Where some rows do not see a position its value must not reach them, whatever it is (zero times an infinity is none): int4 pages' scales and
            // zero points that are not finite are replaced, and the rows that do see them become NaN, as their products would.
            u32 odd = 0;
            if (!F16 && !whole) {
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const u32 w = f.vp[k >> 2][k & 3];
                    const bool strange = (w & 0x7C00u) == 0x7C00u || (w & 0x7C000000u) == 0x7C000000u;
                    odd |= (strange ? 1u : 0u) << k;
                    f.vp[k >> 2][k & 3] = strange || !(ok.ok >> k & 1) ? kNoParameters : w;
                }
                odd &= ok.ok;
            }
            f32x4 x[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) x[nb][0] = x[nb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f16x8 k = __builtin_bit_cast(f16x8, F16 ? f.k[4 * kb + i] : codes_of(f.k[kb][i]));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                        x[nb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, __builtin_bit_cast(f16x8, qf[nb][i]), x[nb][kb], 0, 0, 0);
                }
            u32 keys[8];                                   // {scale, zero} of the keys
#pragma unroll
            for (int k = 0; k < 8; ++k) keys[k] = F16 ? 0u : f.kp[F16 ? 0 : k >> 2][k & 3];
            __builtin_amdgcn_sched_barrier(0);
            there = fetch_keys(next);
            __builtin_amdgcn_sched_barrier(0);
            float vr[8], vz[8];                            // 1 / f and zero point / f of the values
            u32 factors[4], power[4];
            bool plain = true;
            if (!F16) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const u32 w0 = f.vp[k >> 1][2 * k & 3], w1 = f.vp[k >> 1][(2 * k & 3) + 1];
                    power[k] = powers_of(w0, w1, plain);
                    factors[k] = (__builtin_amdgcn_perm(w1, w0, 0x05040100u) & 0x83FF83FFu) | 0x3C003C00u;
                }
                plain = __builtin_amdgcn_ballot_w64(!plain) == 0;
                if (__builtin_expect(!plain, 0)) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float s0 = (float)as_f16x2(f.vp[k >> 1][2 * k & 3])[0], s1 = (float)as_f16x2(f.vp[k >> 1][(2 * k & 3) + 1])[0];
                        factors[k] = cvt_f16x2(factor_of(s0, power_of(s0)), factor_of(s1, power_of(s1)));
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    vr[k] = __builtin_amdgcn_rcpf((float)as_f16x2(factors[k >> 1])[k & 1]);
                    vz[k] = __builtin_fmaf((float)as_f16x2(f.vp[k >> 2][k & 3])[1], vr[k], 0.f);
                }
            }
            u32x4 p[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float y[8], top = -__builtin_inff();
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const f16x2 kp = as_f16x2(keys[k]);
                    y[k] = F16 ? x[nb][k >> 2][k & 3] : __builtin_fmaf(x[nb][k >> 2][k & 3], (float)kp[0], (float)kp[1] * qsum[nb]);
                }
                if (!whole) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] = sees(nb, k) ? y[k] : -__builtin_inff();
                    if (!F16 && __builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) != 0, 0)) {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if ((odd >> k & 1) && sees(nb, k)) d[nb] = __builtin_nanf("");
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) top = __builtin_fmaxf(top, y[k]);
                top *= kUnit;
                if (__builtin_amdgcn_ballot_w64(top > m[nb] + kGrow)) {
                    const float high = quarters_max(top), now = high > m[nb] + kGrow ? high : m[nb], keep = __builtin_amdgcn_exp2f(m[nb] - now);      // (of the row alone)
                    m[nb] = now;
                    d[nb] *= keep, pz[nb] *= keep;
#pragma unroll
                    for (int k = 0; k < 8; ++k) acc[nb][k] *= keep;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[2 * k], kUnit, -m[nb])), w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(y[2 * k + 1], kUnit, -m[nb]));
                    const u32 w = F16 ? cvt_f16x2(w0, w1) : scaled_pair(w0, w1, factors[k]);
                    p[nb][k] = w;
                    const f16x2 r = as_f16x2(w);
                    d[nb] = F16 ? d[nb] + (float)r[0] : __builtin_fmaf((float)r[0], vr[2 * k], d[nb]);
                    d[nb] = F16 ? d[nb] + (float)r[1] : __builtin_fmaf((float)r[1], vr[2 * k + 1], d[nb]);
                    if (!F16) pz[nb] = __builtin_fmaf((float)r[1], vz[2 * k + 1], __builtin_fmaf((float)r[0], vz[2 * k], pz[nb]));
                }
            }
            // the values: row m of block b is dimension 8 m + b
            if (F16) {
                auto product = [&](auto&& word, auto&& add) {      // word(key, word of its piece); add(block, operand)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        u32x4 v[2];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const u32 w0 = word(2 * k, i), w1 = word(2 * k + 1, i);
                            v[0][k] = __builtin_amdgcn_perm(w1, w0, 0x05040100u);
                            v[1][k] = __builtin_amdgcn_perm(w1, w0, 0x07060302u);
                        }
                        add(2 * i, v[0]);
                        add(2 * i + 1, v[1]);
                    }
                };
                auto add_all = [&](int block, u32x4 v) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
                        acc[nb][block] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, v), __builtin_bit_cast(f16x8, p[nb]), acc[nb][block], 0, 0, 0);
                };
                // (opaque to the compiler, which would keep all masks of the loop below in registers)
                auto strange = [](u32 w) {
                    asm volatile("" : "+v"(w));
                    return ((w & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u) | ((w & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u);
                };
                bool any = false;
                if (!whole) {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            f.v4[k][i] = (ok.ok >> k & 1) ? (u32)f.v4[k][i] : 0u;
                            any = any || strange(f.v4[k][i]) != 0;
                        }
                }
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(any) == 0, 1)) {
                    product([&](int k, int i) { return (u32)f.v4[k][i]; }, add_all);
                } else {
                    // infinities and NaN where not all rows see all positions: first all other values, then position by position the rest, for the rows that see it
                    product([&](int k, int i) { return (u32)f.v4[k][i] & ~strange(f.v4[k][i]); }, add_all);
#pragma unroll 1
                    for (int j = 0; j < 32; ++j) {
                        const int pos = at + j;
                        product([&](int k, int i) { return 16 * (k >> 2) + 4 * g + (k & 3) == j ? (u32)f.v4[k][i] & strange(f.v4[k][i]) : 0u; },
                                [&](int block, u32x4 v) {
#pragma unroll
                                    for (int nb = 0; nb < NB; ++nb) {
                                        const bool seen = pos <= place[nb] && (a.window == 0 || pos > place[nb] - a.window || pos < a.sinks);
                                        const f32x4 more = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, v), __builtin_bit_cast(f16x8, p[nb]), f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                                        for (int i = 0; i < 4; ++i) acc[nb][block][i] += seen ? more[i] : 0.f;
                                    }
                                });
                    }
                }
            } else {
                auto product = [&](auto&& scaled) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {     // nibbles 4 half .. 4 half + 3
                        u32x4 v[4];                        // [block][pair of keys]
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const u32x4 w = scaled(__builtin_amdgcn_perm(f.v[2 * k + 1], f.v[2 * k], half ? 0x07060302u : 0x05040100u), k);
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[i][k] = w[i];
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb)
                                acc[nb][4 * half + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, v[i]), __builtin_bit_cast(f16x8, p[nb]), acc[nb][4 * half + i], 0, 0, 0);
                    }
                };
                if (__builtin_expect(plain, 1)) product([&](u32 w, int k) { return scaled_codes(w, power[k], masks); });
                else product([&](u32 w, int k) { return scaled_codes_slow(w, f.vp[k >> 1][2 * k & 3], f.vp[k >> 1][(2 * k & 3) + 1]); });
            }
        };

        for (; s < steps.all; s += stride) {
            const int next = s + stride < steps.all ? s + stride : s;  // (behind the last step the next one is the same again)
            if (ALIGNED && next != s && ++turn == 32) fetch_pages(next);
            consume(s, next);
            __builtin_amdgcn_sched_barrier(0);
            fetch_values();
            __builtin_amdgcn_sched_barrier(0);
        }

        // ---- merge: a wave's states are those of its rows; the waves' through LDS, one block of 16 rows at a time
        constexpr int LANES = NW < 8 ? 4 * NW : 32, PER = 32 / LANES;        // threads of a row, and of its 32 pieces of four dimensions how many each takes
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const float dd = quarters_sum(d[nb]), zz = F16 ? 0.f : quarters_sum(pz[nb]);
            __syncthreads();
            f32x4* const mine = st4 + (wave * 16 + n) * 33;
            if (g == 0) mine[0] = f32x4{m[nb], dd, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {                  // dimensions 8 (4 g + i) + block
                mine[1 + 8 * g + 2 * i] = f32x4{acc[nb][0][i] - zz, acc[nb][1][i] - zz, acc[nb][2][i] - zz, acc[nb][3][i] - zz};
                mine[2 + 8 * g + 2 * i] = f32x4{acc[nb][4][i] - zz, acc[nb][5][i] - zz, acc[nb][6][i] - zz, acc[nb][7][i] - zz};
            }
            __syncthreads();
            const int row = threadIdx.x / LANES, l = threadIdx.x % LANES, r = r0 + 16 * nb + row;
            if (row < 16 && r < rows) {
                float M = kEmpty, D = 0.f;
#pragma unroll
                for (int w = 0; w < NW; ++w) M = __builtin_fmaxf(M, st4[(w * 16 + row) * 33][0]);
                f32x4 O[PER];
#pragma unroll
                for (int i = 0; i < PER; ++i) O[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < NW; ++w) {
                    const f32x4* src = st4 + (w * 16 + row) * 33;
                    const float keep = __builtin_amdgcn_exp2f(src[0][0] - M);
                    D = __builtin_fmaf(src[0][1], keep, D);
#pragma unroll
                    for (int i = 0; i < PER; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) O[i][j] = __builtin_fmaf(src[1 + PER * l + i][j], keep, O[i][j]);
                }
                const int t = divided(r, a.per_group), head = h * a.group + r - t * a.group;
                bool finished = a.splits == 1;
                if constexpr (SHARED) finished = !a.states;
                if (finished) {
                    if constexpr (SHARED) {
                        if (a.join > 0 && (!a.members || (a.first + b >= a.members[0] && a.first + b < a.members[a.prefixes]))) {
                            // the states of the prefix that the row's sequence shares
                            const f32x4* const src = (const f32x4*)a.part + ((int64_t)(start + t) * (c.num_heads * a.group) + head) * a.join * 33;
                            for (int from = 0; from < a.join; from += 4) {
                                f32x4 state[4], x[4][PER];
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const f32x4* const at = src + (from + i < a.join ? from + i : a.join - 1) * 33;
                                    state[i] = at[0];
#pragma unroll
                                    for (int j = 0; j < PER; ++j) x[i][j] = at[1 + PER * l + j];
                                }
                                float high = M;
#pragma unroll
                                for (int i = 0; i < 4; ++i) high = __builtin_fmaxf(high, state[i][0]);
                                const float mine = __builtin_amdgcn_exp2f(M - high);
                                M = high, D *= mine;
#pragma unroll
                                for (int j = 0; j < PER; ++j) O[j] *= mine;
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    // (an empty state may be its maximum and sum alone: what lies behind them is anything)
                                    const bool is = from + i < a.join && state[i][0] != kEmpty;
                                    const float keep = is ? __builtin_amdgcn_exp2f(state[i][0] - high) : 0.f;
                                    D += is ? state[i][1] * keep : 0.f;
#pragma unroll
                                    for (int j = 0; j < PER; ++j) O[j] += is ? x[i][j] * keep : f32x4{0.f, 0.f, 0.f, 0.f};
                                }
                            }
                        }
                    }
                    const float inv = D == 0.f ? 0.f : 1.f / D;                 // (a row that sees nothing is zero)
                    if constexpr (SHARED)
                        if (a.lse && l == 0) a.lse[(int64_t)(start + t) * (c.num_heads * a.group) + head] = lse_of(M, D);
                    u32x2* const dst = (u32x2*)(a.o + (int64_t)(start + t) * a.o_stride + (int64_t)head * 128) + PER * l;
#pragma unroll
                    for (int i = 0; i < PER; ++i) dst[i] = u32x2{cvt_f16x2(O[i][0] * inv, O[i][1] * inv), cvt_f16x2(O[i][2] * inv, O[i][3] * inv)};
                } else {
                    int parts = a.splits, at = split;
                    if constexpr (SHARED) parts = a.parts, at = a.part_at + split;
                    float* dst = a.part + (((int64_t)(start + t) * (c.num_heads * a.group) + head) * parts + at) * 132;
                    if (l == 0) dst[0] = M, dst[1] = D;
#pragma unroll
                    for (int i = 0; i < PER; ++i) *((f32x4*)dst + 1 + PER * l + i) = O[i];
                }
            }
        }
    }
}

template <int NB, int NW, bool F16, bool ALIGNED, bool SHARED>
__global__ __launch_bounds__(64 * NW, NB == 2 || F16 ? 2 : 3) void chunk_rows_kernel(Launch<SHARED> a, Divisor pages) { attend_rows<NB, NW, F16, ALIGNED, SHARED>(a, pages, blockIdx.x); }
// Two launches in one: the first `groups` workgroups are a's, the others b's
template <bool F16, bool ALIGNED>
__global__ __launch_bounds__(256, F16 ? 2 : 3) void chunk_rows_pair_kernel(Chunk a, Chunk b, Divisor pages, int groups) {
    const bool first = (int)blockIdx.x < groups;
    attend_rows<1, 4, F16, ALIGNED, true>(first ? a : b, pages, first ? blockIdx.x : blockIdx.x - groups);
}

// The partial states of every row -> its output: sixteen lanes per row, eight dimensions each.  The states' maxima and sums are read by a lane each (at most 32),
// so that all loads are on their way at once: with few rows this launch is their latency (64 rows of 32 states: 5.6 us; with the states read one after the other 20.3).
__global__ __launch_bounds__(64) void chunk_merge_kernel(const float* __restrict__ part, const int32_t* __restrict__ starts, int batch, int tokens,
                                                          int heads, Divisor per_head, int splits, f16* __restrict__ o, int64_t o_stride) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 4);
    const int l = threadIdx.x & 15;
    const int64_t token = divided((int)row, per_head);     // (rows are fewer than 2^30)
    const int head = (int)(row - token * heads);
    // (rows that belong to no sequence have no states and are left as they are)
    if (token >= tokens || (starts && (token < starts[0] || token >= starts[batch]))) return;
    const f32x4* src = (const f32x4*)(part + row * splits * 132);
    const f32x4 none = {kEmpty, 0.f, 0.f, 0.f};
    const f32x4 first = l < splits ? src[l * 33] : none, second = l + 16 < splits ? src[(l + 16) * 33] : none;
    float M = __builtin_fmaxf(first[0], second[0]);
#pragma unroll
    for (int bit = 1; bit < 16; bit *= 2) M = __builtin_fmaxf(M, __shfl_xor(M, bit, 16));
    const float keep[2] = {__builtin_amdgcn_exp2f(first[0] - M), __builtin_amdgcn_exp2f(second[0] - M)};
    float D = __builtin_fmaf(first[1], keep[0], second[1] * keep[1]);
#pragma unroll
    for (int bit = 1; bit < 16; bit *= 2) D += __shfl_xor(D, bit, 16);
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    for (int from = 0; from < splits; from += 8) {
        f32x4 x[8], y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int s = from + i < splits ? from + i : splits - 1;
            x[i] = src[s * 33 + 1 + 2 * l], y[i] = src[s * 33 + 2 + 2 * l];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float k = __shfl(from < 16 ? keep[0] : keep[1], (from + i) & 15, 16);
            if (from + i < splits) {
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = __builtin_fmaf(x[i][j], k, a[j]), b[j] = __builtin_fmaf(y[i][j], k, b[j]);
            }
        }
    }
    const float inv = D == 0.f ? 0.f : 1.f / D;
    *((u32x4*)(o + token * o_stride + (int64_t)head * 128) + l) =
        u32x4{cvt_f16x2(a[0] * inv, a[1] * inv), cvt_f16x2(a[2] * inv, a[3] * inv), cvt_f16x2(b[0] * inv, b[1] * inv), cvt_f16x2(b[2] * inv, b[3] * inv)};
}

// The same where a row's states are of two launches, `own` of its sequence's positions and then those of the prefix that its sequence shares (a row of a sequence
// outside members[0] .. members[prefixes] has none of these), and where the logarithms of the sums are asked for.
struct Joined {
    const float* part;
    const int32_t *starts, *members;
    f16* o;
    float* lse;                        // may be nullptr
    int64_t o_stride;
    int batch, tokens, heads, prefixes, own, parts;
    Divisor per_head;
};
// QUARTERS 4: a wave per row, whose quarters take every fourth state, so that the states of a row that has many are on their way at once (256 rows
// of 34 states: a call of 27.0 us takes 23.1); 1: four rows per wave, for many rows (139264 of three states: 41 us, with a wave each 86).
template <int QUARTERS>
__global__ __launch_bounds__(256) void chunk_join_kernel(Joined a) {
    const int64_t row = (int64_t)blockIdx.x * (16 / QUARTERS) + (threadIdx.x / (16 * QUARTERS));
    const int l = threadIdx.x & 15, quarter = QUARTERS == 4 ? threadIdx.x >> 4 & 3 : 0;
    const int token = divided((int)row, a.per_head), head = (int)row - token * a.heads;
    if (token >= a.tokens || (a.starts && (token < a.starts[0] || token >= a.starts[a.batch]))) return;
    int from_token = 0, to_token = 0x7fffffff;             // tokens of sequences that have a prefix
    if (a.members) {
        auto bound = [&](int i) {
            const int s = a.members[i], in = s < 0 ? 0 : s > a.batch ? a.batch : s;
            return a.starts ? a.starts[in] : in;
        };
        from_token = bound(0), to_token = bound(a.prefixes);
    }
    const int states = token >= from_token && token < to_token ? a.parts : a.own;
    const f32x4* const src = (const f32x4*)(a.part + row * a.parts * 132);
    constexpr int EACH = 4;                                // states of a quarter at a time
    float M = kEmpty, D = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
    for (int from = 0; from < states; from += QUARTERS * EACH) {
        f32x4 head4[EACH], x4[EACH], y4[EACH];
        float high = M;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int s = from + QUARTERS * i + quarter;
            const f32x4* const at = src + (s < states ? s : states - 1) * 33;
            head4[i] = at[0], x4[i] = at[1 + 2 * l], y4[i] = at[2 + 2 * l];
            if (s >= states) head4[i][0] = kEmpty;
        }
#pragma unroll
        for (int i = 0; i < EACH; ++i) high = __builtin_fmaxf(high, head4[i][0]);
        const float mine = __builtin_amdgcn_exp2f(M - high);
        M = high, D *= mine;
        x *= mine, y *= mine;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const bool is = head4[i][0] != kEmpty;         // (an empty state may be its maximum and sum alone: what lies behind them is anything)
            const float keep = is ? __builtin_amdgcn_exp2f(head4[i][0] - high) : 0.f;
            D += is ? head4[i][1] * keep : 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] += is ? x4[i][j] * keep : 0.f, y[j] += is ? y4[i][j] * keep : 0.f;
        }
    }
    if (QUARTERS == 4) {
        const float all = quarters_max(M), mine = __builtin_amdgcn_exp2f(M - all);
        M = all, D = quarters_sum(D * mine);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = quarters_sum(x[j] * mine), y[j] = quarters_sum(y[j] * mine);
        if (quarter) return;
    }
    const float inv = D == 0.f ? 0.f : 1.f / D;
    if (a.lse && l == 0) a.lse[row] = lse_of(M, D);
    *((u32x4*)(a.o + (int64_t)token * a.o_stride + (int64_t)head * 128) + l) =
        u32x4{cvt_f16x2(x[0] * inv, x[1] * inv), cvt_f16x2(x[2] * inv, x[3] * inv), cvt_f16x2(y[0] * inv, y[1] * inv), cvt_f16x2(y[2] * inv, y[3] * inv)};
}

// How a call is cut: column blocks and waves of a workgroup (nb 0: the kernel of 256 rows), tiles of rows per (sequence, key head), splits of the
// positions.
//
// (Microseconds of sequences of one length, median of calls back to back.)  16 rows and fewer read the cache once, whoever does it.  Int4 pages: twelve waves to a
// compute unit, in one workgroup where there are sequences and heads enough, or little to read (one token, 64 on 8 heads: 32 x 4096 33, 8 waves 35, 4 waves 41;
// 32 x 500 11.0, 10.9 and 10.8; where two such workgroups follow one another on a compute unit 4 waves are ahead, 64 x 2000 39.5, 38.5 and 32.5, which the rule
// does not go by), else in three, split (4 x 4000, 32 heads: 22.5; 8 waves, split in two 22.5; 12 waves 29), or one with the most splits there are (30000, 64 on 8
// heads: 21.4; 4 waves 21.0, in 24 splits 22.1).  Fp16 pages have registers for two workgroups of four waves (64 x 1000, 32 heads: 189 us, 5.5 TB/s; one of eight
// 203; 2000: 14.5 in 7 splits, 16.0 of 8 waves in 4).
//
// More rows are a choice between tiles of 32, each of which reads and unpacks the cache for itself, and tiles of 256, whose workgroups have a
// compute unit to themselves and a long way to their first product.  Microseconds, from the two kernels' own times: a wave's step of 32
// positions by 32 rows 2.4 with two waves per SIMD (fp16 pages, which reach the caches' bandwidth, 5.5), 6.5 around them; a step of 64
// positions by 256 rows 2.9, 14 around them; partial states 0.17 a thousand, and 6 for one more launch.  The cut of the least sum is taken.
// Measured, tiles of 32 and of 256, each at its best (4000 tokens cached, 32 heads, int4): 192 rows 46 and 50 us, 8 x 96 119 and 162, 8 x 128 151 and 171,
// 8 x 192 222 and 179, 8 x 256 293 and 186; 500 cached: 256 rows 17 and 32, 8 x 256 74 and 52; fp16 pages: 8 x 64 162 and 175, 8 x 96 326
// and 181.  Splits of tiles of 256: 512 rows after 4001 119, 89, 77, 103 with 2, 3, 4, 6.  (64 rows per wave of the small kernel, at one wave
// per SIMD, were slower than 32 everywhere, by up to 3 times.)
//
// Partial states fill at most kMostParts bytes: a call of that many rows (16384 tokens of 64 heads in two splits) has 16 turns of tiles of 256 and more, and a split
// gains no more than a part of the last one.
struct ChunkPlan {
    int nb, nw, tiles, splits, dealt = 0;
};
constexpr size_t kMostParts = (size_t)1 << 30;
constexpr int kMostHeads = 65536;                          // (with most splits a sequence's heads are a launch)
size_t part_bytes(int64_t tokens, int64_t q_heads, int parts) { return (size_t)tokens * q_heads * parts * 132 * sizeof(float); }
size_t chunk_part_bytes(int64_t tokens, int64_t q_heads, int splits) { return splits > 1 ? part_bytes(tokens, q_heads, splits) : 0; }
ChunkPlan chunk_plan(bool fp16, int64_t tokens, int group, int num_heads, int64_t batch, int64_t max_new_len, int64_t max_seq_len, int64_t window, int64_t sinks) {
    if (max_new_len <= 0 || max_new_len > tokens) max_new_len = tokens;
    if (max_new_len < (tokens + batch - 1) / batch) max_new_len = (tokens + batch - 1) / batch;        // (some sequence has as many)
    const bool even = max_new_len * batch == tokens;
    const int64_t rows = max_new_len * group, cus = qr_device().cus;
    int64_t seen = max_seq_len < 0 ? 0 : max_seq_len < 0x3fffffff ? max_seq_len : 0x3fffffff;              // (no sequence is as long)
    window = window < 0x3fffffff ? window : 0x3fffffff, sinks = sinks < 0x3fffffff ? sinks : 0x3fffffff;
    if (window > 0 && window < seen && sinks < seen && seen > window + max_new_len + sinks + 64) seen = window + max_new_len + sinks + 64;
    ChunkPlan p{1, 4, 1, 1};
    if (rows <= 16) {
        const int64_t groups = batch * num_heads, steps = (seen + 31) / 32;
        int64_t splits = 1;
        if (fp16) {
            if (groups < cus) splits = (2 * cus + groups - 1) / groups;
            if (splits > steps / 8) splits = steps / 8;                          // (two steps per wave at least)
        } else if (groups >= cus || steps <= 24) {
            p.nw = steps <= 8 ? 4 : 12;
        } else if (32 * groups >= 3 * cus) {
            splits = (3 * cus + groups - 1) / groups;
            if (splits > steps / 4) splits = steps / 4;
        } else {
            p.nw = 12;
            splits = steps / 12 < cus / groups ? steps / 12 : cus / groups;
        }
        p.splits = splits < 1 ? 1 : splits > 32 ? 32 : (int)splits;
        return p;
    }
    float least = -1.f;
    auto consider = [&](int nb, int nw, int64_t per, int64_t at_once, int64_t step, float each, float around) {
        const int64_t tiles = (rows + per - 1) / per;
        int64_t groups = batch * tiles;
        if (!even) {                                       // (a ragged batch's tiles are guessed)
            int64_t some = tokens * group / per + batch / 2;
            if (some < batch) some = batch;
            if (some < groups) groups = some;
        }
        groups *= num_heads;
        const int64_t late = max_new_len - per / group;    // (what the first tile does not see of the last one's positions, at most)
        const float steps = (float)(seen - (late > 0 ? (late < seen ? late : seen) / 2 : 0)) / (float)step;
        for (int s = 1; s <= 32; ++s) {
            if (s > 1 && (steps < (float)(3 * s) || chunk_part_bytes(tokens, (int64_t)group * num_heads, s) > kMostParts)) break;
            const float turns = (float)((int64_t)(steps / (float)s) + 1);
            const float time = (float)((groups * s + at_once - 1) / at_once) * (turns * each + around) +
                               (s > 1 ? 6.f + (float)(tokens * group * num_heads) * (float)s * (660.f / 4e6f) : 0.f);
            if (least < 0.f || time < least) least = time, p = ChunkPlan{nb, nw, (int)(tiles > 4096 ? 4096 : tiles), s};       // (a workgroup goes on to the next tile behind them)
        }
    };
    const float small = fp16 ? 5.5f : 2.4f;
    consider(2, 8, 32, cus, 32 * 8, small, 6.5f);
    consider(2, 4, 32, 2 * cus, 32 * 4, small, 6.5f);
    consider(0, 4, 256, cus, 64, 2.9f, 14.f);
    return p;
}

template <bool F16, bool ALIGNED, bool SHARED>
int launch_rows(const ChunkPlan& plan, const Chunk& a, Divisor pages, int64_t groups, hipStream_t st) {
    using Kernel = void (*)(Launch<SHARED>, Divisor);
    const Kernel kernel = plan.nb == 2 ? (plan.nw == 8 ? chunk_rows_kernel<2, 8, F16, ALIGNED, SHARED> : chunk_rows_kernel<2, 4, F16, ALIGNED, SHARED>)
                                       : (F16 || plan.nw == 4 ? chunk_rows_kernel<1, 4, F16, ALIGNED, SHARED> : chunk_rows_kernel<1, F16 ? 4 : 12, F16, ALIGNED, SHARED>);
    const size_t lds = (size_t)plan.nw * 16 * 33 * sizeof(f32x4);
    const hipError_t e = qr_allow_dynamic_lds((const void*)kernel, lds);
    if (e != hipSuccess) return (int)e;
    kernel<<<dim3((unsigned)groups), dim3(64 * plan.nw), lds, st>>>(a, pages);
    return qr_launch_status();
}

// The launches of one set of page tables: a's sequences (or prefixes) as the plan cuts them.  A launch has fewer than 2^32 threads: fewer tiles at a time where hints
// are missing (a workgroup goes on to the next one behind them), then fewer sequences.
template <bool SHARED>
int launch_chunk(bool fp16, const ChunkPlan& plan, Chunk a, hipStream_t st) {
    const int64_t batch_size = a.c.batch_size, num_q_heads = (int64_t)a.c.num_heads * a.group;
    a.tiles = plan.tiles;
    a.splits = plan.dealt ? 1 : plan.splits, a.per_split = divisor_of(a.splits);
    a.dealt = plan.dealt;
    const int64_t most = 0xffffffffll / (plan.nb == 0 ? 256 : 64 * plan.nw), wide = (int64_t)a.c.num_heads * a.splits;
    if (!a.dealt && batch_size * wide * plan.tiles > most) a.tiles = (int)(batch_size * wide < most ? most / (batch_size * wide) : 1);
    const int64_t at_once = batch_size * wide <= most ? batch_size : most / wide;
    const Divisor pages = divisor_of(a.c.page_size);
    const bool aligned = a.c.page_size % 16 == 0;
    int rc = QR_OK;
    for (int64_t first = 0; first < batch_size && rc == QR_OK; first += at_once) {
        Chunk some = a;
        some.c.batch_size = (int)(batch_size - first < at_once ? batch_size - first : at_once);
        some.c.indptr += first, some.c.last_page_offset += first;
        some.first = (int)first;
        if (a.prefix) some.members += a.members ? first : 0;
        else if (a.starts) some.starts += first;
        else {
            some.q += first * a.q_stride, some.o += first * a.o_stride;
            some.part += a.states ? first * num_q_heads * a.parts * 132 : first * num_q_heads * a.join * 132;
            some.lse += a.lse ? first * num_q_heads : 0;
        }
        const int64_t groups = a.dealt ? a.dealt : some.c.batch_size * wide * a.tiles;
        rc = plan.nb == 0 ? qr_internal_chunk_tiles(fp16, some, pages, groups, st)
             : fp16       ? (aligned ? launch_rows<true, true, SHARED>(plan, some, pages, groups, st) : launch_rows<true, false, SHARED>(plan, some, pages, groups, st))
                          : (aligned ? launch_rows<false, true, SHARED>(plan, some, pages, groups, st) : launch_rows<false, false, SHARED>(plan, some, pages, groups, st));
    }
    return rc;
}

struct ChunkCall {
    void* o;
    int64_t o_stride;
    const void* q;
    int64_t q_stride;
    int q_had_mode;
    const void* starts;
    int64_t tokens;
    int num_q_heads;
    const void *kv_data, *kv_param, *kv_indptr, *kv_indices, *last_page_offset;
    int64_t num_pages;
    int num_layers, layer_idx, num_heads, page_size, head_dim;
    int64_t batch_size, max_new_len, max_seq_len, window, sinks;
    void* workspace;
    size_t workspace_bytes;
    void* stream;
};
int check_chunk(const ChunkCall& t) {
    const int rc = qr_internal_check_paged_cache(t.kv_data, t.kv_param, t.kv_indptr, t.kv_indices, t.last_page_offset, t.num_pages, t.num_layers, t.layer_idx, t.num_heads,
                                                 t.page_size, t.head_dim, t.batch_size);
    if (rc != QR_OK) return rc;
    if (t.q_had_mode != 0 && t.q_had_mode != 1) return QR_E_DTYPE;
    if (t.tokens < 0 || t.num_q_heads <= 0 || t.num_q_heads % t.num_heads || t.window < 0 || t.sinks < 0 || t.max_new_len < 0 || t.max_seq_len < 0) return QR_E_SHAPE;
    if (t.tokens == 0 || t.batch_size == 0) return QR_OK;
    if (!t.starts && t.tokens != t.batch_size) return QR_E_SHAPE;                // one new token per sequence
    if (!t.o || !t.q) return QR_E_NULL;
    if (((uintptr_t)t.q & 15) || ((uintptr_t)t.o & 15) || t.q_stride % 8 || t.o_stride % 8) return QR_E_ALIGN;
    const int64_t width = (int64_t)t.num_q_heads * 128;
    if (t.q_stride < width || t.o_stride < width || t.tokens > 0x3fffffff || t.tokens * t.num_q_heads > 0x3fffffff || t.num_q_heads / t.num_heads > 1024 || t.num_heads > kMostHeads)
        return QR_E_SHAPE;
    return QR_OK;
}
Chunk chunk_of(const ChunkCall& t) {
    Chunk a;
    a.c = qr_internal_paged_kv((void*)t.kv_data, (void*)t.kv_param, t.kv_indptr, t.kv_indices, t.last_page_offset, t.num_pages, t.num_layers, t.layer_idx, t.num_heads,
                               t.page_size, t.batch_size);
    a.q = (const f16*)t.q;
    a.o = (f16*)t.o;
    a.starts = (const int32_t*)t.starts;
    a.q_stride = t.q_stride, a.o_stride = t.o_stride;
    a.tokens = (int)t.tokens;
    a.group = t.num_q_heads / t.num_heads;
    a.per_group = a.per_place = divisor_of(a.group);
    a.per_head = divisor_of(t.num_heads);
    a.window = (int)(t.window > 0x3fffffff ? 0 : t.window);              // (longer than any sequence)
    a.sinks = (int)(t.sinks > 0x3fffffff ? 0x3fffffff : t.sinks);
    a.q_had = t.q_had_mode;
    a.members = nullptr;
    a.dealt = 0, a.prefix = 0, a.sequences = (int)t.batch_size, a.prefixes = 0, a.first = 0, a.join = 0;
    a.part = (float*)t.workspace;
    a.part_at = 0;
    a.lse = nullptr;
    return a;
}
ChunkPlan plan_of(bool fp16, const ChunkCall& t) {
    return chunk_plan(fp16, t.tokens, t.num_q_heads / t.num_heads, t.num_heads, t.batch_size, t.starts ? t.max_new_len : 1, t.max_seq_len, t.window, t.sinks);
}

int batch_chunk(bool fp16, const ChunkCall& t) {
    const int rc = check_chunk(t);
    if (rc != QR_OK || t.tokens == 0 || t.batch_size == 0) return rc;
    ChunkPlan plan = plan_of(fp16, t);
    if (plan.splits > 1 && (!t.workspace || ((uintptr_t)t.workspace & 15) || t.workspace_bytes < chunk_part_bytes(t.tokens, t.num_q_heads, plan.splits))) plan.splits = 1;
    Chunk a = chunk_of(t);
    a.parts = plan.splits, a.states = plan.splits > 1;
    hipStream_t st = (hipStream_t)t.stream;
    const int lrc = launch_chunk<false>(fp16, plan, a, st);
    if (lrc != QR_OK || plan.splits == 1) return lrc;
    chunk_merge_kernel<<<dim3((unsigned)((t.tokens * t.num_q_heads + 3) / 4)), dim3(64), 0, st>>>(a.part, a.starts, (int)t.batch_size, (int)t.tokens, t.num_q_heads,
                                                                                                  divisor_of(t.num_q_heads), plan.splits, a.o, t.o_stride);
    return qr_launch_status();
}

// ---- prefixes that several sequences share ---------------------------------------------------------------------------------------------------
// A prefix is a page list that is attended to by the rows of all its sequences' tokens, as if they were one sequence's that see all of it: its vectors are read (and
// unpacked) once per tile of those rows instead of once per sequence.  A row's states of both launches are joined by the sequences' own launch, or by a third; where both are tiles
// of 16 rows they are one launch.
// (4 of 101 after 1200, 32 heads: 12.0 us, two launches; 64 of up to 701 after 8192, 64 on 8 heads: 58, of which 42 are the prefix's tiles, 12 of these before and behind their eight
// steps, and 16 the sequences' with 35 MB of states; fp16 pages, 30 of up to 338 after three of 2999, 40 heads: 68.5, 3.4 TB/s; 16 of up to 256 new after 16384, 64 on 8 heads:
// 1400 - 1440, 815 - 837 TFLOP/s.)
//
// How the prefixes' launch is cut: tiles of 16, 32 or 256 rows, and splits of the positions, whose states are written in any case.  The cut of the least sum is taken,
// of the kernels' own times in microseconds: a step of a wave (32 positions by 16 or 32 rows, shorter where the chip is not full) or of a workgroup
// (64 by 256), what goes around the steps, 0.16 a thousand states.  The numbers are those that lose least over 16 .. 1024 rows of 8 and 32 key heads after
// 500 .. 24000 positions, 1 - 2 % on average against the best of 5 to 40 cuts (the rule above, which knows no tiles of 16 of more than 16 rows and counts a
// third launch: 10 - 13 %).  Int4 pages, microseconds of a whole call with tiles of 16, 32 and 256, each at its best: 64 rows of 8 heads after 2000 17.2,
// 19.7, 28.3; after 24000 36.6, 33.7, 54.2; 512 rows after 8000 -, 54.0, 53.3; after 24000 -, 121, 90.5.  Fp16 pages: 64 rows after 8000 26.2, 32.3, 36.7;
// 256 rows -, 49.3, 44.7.
ChunkPlan prefix_plan(bool fp16, int64_t tokens, int group, int num_heads, int64_t prefixes, int64_t max_len) {
    const int64_t rows = tokens * group, cus = qr_device().cus, seen = max_len < 0x3fffffff ? max_len : 0x3fffffff;
    ChunkPlan p{1, 4, 1, 1};
    float least = -1.f;
    auto consider = [&](int nb, int nw, int64_t per, int64_t at_once, int64_t step, float each, float around, float part, float each_state) {
        int64_t some = prefixes == 1 ? (rows + per - 1) / per : rows / per + prefixes / 2;
        if (some < prefixes) some = prefixes;
        const int64_t groups = some * num_heads, most = (rows + per - 1) / per, even = 3 * ((rows + prefixes * per - 1) / (prefixes * per)), steps = (seen + step - 1) / step;
        for (int s = 1; s <= 32; ++s) {
            if (s > 1 && (steps < s || chunk_part_bytes(tokens, (int64_t)group * num_heads, s) > kMostParts)) break;
            const float turns = (float)((steps + s - 1) / s), full = (float)(groups * s) / (float)at_once;
            const float time = (float)((groups * s + at_once - 1) / at_once) * (turns * each * (part + (1.f - part) * (full < 1.f ? full : 1.f)) + around) +
                               (float)(rows * num_heads) * (float)s * each_state;
            const int64_t tiles = most < even ? most : even;               // (a workgroup goes on to the next tile behind them)
            if (least < 0.f || time < least) least = time, p = ChunkPlan{nb, nw, (int)(tiles > 4096 ? 4096 : tiles), s};
        }
    };
    // One prefix: the steps of all its tiles in equal shares (qr_deal.h).
    auto deal = [&](float each, float around, float part, float each_state) {
        int64_t tiles = (rows + 255) / 256;
        tiles = tiles > 4096 ? 4096 : tiles;               // (rows are fewer than 2^30; what lies behind is left to the splits of whole tiles)
        if (tiles * 256 < rows) return consider(0, 4, 256, cus, 64, each, around, part, each_state);
        const int64_t all = tiles * num_heads, steps = (seen + 63) / 64 < 1 ? 1 : (seen + 63) / 64;
        const DealtCut cut = dealt_cut(all, seen > 0 ? steps : 0, cus);
        const int64_t shares = cut.shares, states = cut.states;
        const float full = (float)shares / (float)cus;
        const float time = (float)(all * steps + shares - 1) / (float)shares * each * (part + (1.f - part) * (full < 1.f ? full : 1.f)) +
                           (float)((all + shares - 1) / shares + (all % shares && shares % all ? 1 : 0)) * around + (float)(rows * num_heads) * (float)states * each_state;
        if (chunk_part_bytes(tokens, (int64_t)group * num_heads, (int)states) > kMostParts && states > 2) return consider(0, 4, 256, cus, 64, each, around, part, each_state);
        if (least < 0.f || time < least) least = time, p = ChunkPlan{0, 4, (int)tiles, (int)states, (int)shares};
    };
    const bool few = rows <= 64 * prefixes;                // (the tiles of 16 were measured up to there)
    if (fp16) {
        if (few) consider(1, 4, 16, cus, 32 * 4, 0.87f, 4.7f, 0.6f, 1.75e-4f);
        consider(2, 4, 32, 2 * cus, 32 * 4, 5.3f, 6.5f, 0.6f, 1.75e-4f);
        consider(2, 8, 32, cus, 32 * 8, 5.3f, 7.3f, 0.6f, 1.75e-4f);
        if (prefixes > 1) consider(0, 4, 256, cus, 64, 3.27f, 14.f, 0.6f, 1.75e-4f);
        else deal(3.27f, 14.f, 0.6f, 1.75e-4f);
    } else {
        if (few) consider(1, 4, 16, 3 * cus, 32 * 4, 0.72f, 4.7f, 0.46f, 1.62e-4f);
        consider(2, 4, 32, 2 * cus, 32 * 4, 2.4f, 6.5f, 0.46f, 1.62e-4f);
        consider(2, 8, 32, cus, 32 * 8, 2.4f, 7.7f, 0.46f, 1.62e-4f);
        if (prefixes > 1) consider(0, 4, 256, cus, 64, 2.9f, 8.1f, 0.46f, 1.62e-4f);
        else deal(2.9f, 8.1f, 0.46f, 1.62e-4f);
    }
    return p;
}

struct Prefixes {
    const void *indptr, *indices, *last_page_offset, *members;
    int64_t count, max_len;
};
struct SharedPlan {
    ChunkPlan own, prefix;
    int parts;                         // states per row; 1: none are written
    bool paired;                       // both are tiles of 16 rows and one launch
    bool joined;                       // the sequences' own launch takes the prefixes' states in, so that it has none and there is no third launch
};
SharedPlan shared_plan(bool fp16, const ChunkCall& t, int64_t prefixes, int64_t max_prefix_len) {
    SharedPlan p{plan_of(fp16, t), ChunkPlan{0, 0, 0, 0}, 0, false, false};
    if (prefixes > 0) {
        p.prefix = prefix_plan(fp16, t.tokens, t.num_q_heads / t.num_heads, t.num_heads, prefixes, max_prefix_len);
        // (int4 pages, 64 sequences of up to 700 positions of their own, 64 on 8 heads: 16.7 us, with twelve waves 22.5)
        if (p.own.nb == 1 && p.own.nw == 12 && t.batch_size * t.num_heads >= 2 * qr_device().cus) p.own.nw = 4;
        p.paired = p.own.nb == 1 && p.prefix.nb == 1;
        if (p.paired) {
            // Each has a workgroup to a CU where two turns of its four waves' steps make as many.  (Prefix and own splits, microseconds cold: 8 sequences of 300 after 4000, 64 on
            // 8 heads 8 and 2 15.2, 12 and 2 16.4, 3 and 1 18.0; one of 3000 after 300, 32 heads 2 and 8 14.2, 2 and 4 16.4, 2 and 16 15.3.  One launch instead of two:
            // 4 of 100 after 1200, 32 heads 15.7 -> 12.5; fp16 pages, 30 of up to 333 behind three prefixes 85 -> 68.)
            const int64_t cus = qr_device().cus, heads = t.num_heads, group = t.num_q_heads / t.num_heads;
            auto cut = [&](int64_t groups, int64_t positions) {
                const int64_t steps = (positions + 31) / 32, turns = (steps + 7) / 8;
                int64_t s = groups < cus ? cus / groups : 1;
                s = s < turns ? s : turns;
                return (int)(s < 1 ? 1 : s > 32 ? 32 : s);
            };
            const int64_t tiles = prefixes == 1 ? (t.tokens * group + 15) / 16 : t.tokens * group / 16 + prefixes / 2;
            p.own.nw = 4, p.own.splits = cut(t.batch_size * heads, t.max_seq_len < 0x3fffffff ? t.max_seq_len : 0x3fffffff);
            p.prefix.splits = cut((tiles < prefixes ? prefixes : tiles) * heads, max_prefix_len < 0x3fffffff ? max_prefix_len : 0x3fffffff);
            const int64_t most = (int64_t)(0xffffffffll / 256);                // (one launch)
            if (t.batch_size * heads * p.own.splits + prefixes * heads * p.prefix.splits * p.prefix.tiles > most) p.paired = false;
        }
        p.joined = !p.paired && p.own.splits == 1 && p.own.nb != 0;
    }
    p.parts = (p.joined ? 0 : p.own.splits) + p.prefix.splits;
    return p;
}

int launch_pair(bool fp16, const SharedPlan& plan, Chunk prefix, Chunk own, hipStream_t st) {
    prefix.tiles = plan.prefix.tiles, prefix.splits = plan.prefix.splits, prefix.per_split = divisor_of(plan.prefix.splits);
    own.tiles = plan.own.tiles, own.splits = plan.own.splits, own.per_split = divisor_of(plan.own.splits), own.states = 1;
    const int64_t first = (int64_t)prefix.c.batch_size * prefix.c.num_heads * prefix.splits * prefix.tiles;
    const int64_t second = (int64_t)own.c.batch_size * own.c.num_heads * own.splits * own.tiles;
    using Kernel = void (*)(Chunk, Chunk, Divisor, int);
    const bool aligned = own.c.page_size % 16 == 0;
    const Kernel kernel = fp16 ? (aligned ? chunk_rows_pair_kernel<true, true> : chunk_rows_pair_kernel<true, false>)
                               : (aligned ? chunk_rows_pair_kernel<false, true> : chunk_rows_pair_kernel<false, false>);
    const size_t lds = (size_t)4 * 16 * 33 * sizeof(f32x4);
    const hipError_t e = qr_allow_dynamic_lds((const void*)kernel, lds);
    if (e != hipSuccess) return (int)e;
    kernel<<<dim3((unsigned)(first + second)), dim3(256), lds, st>>>(prefix, own, divisor_of(own.c.page_size), (int)first);
    return qr_launch_status();
}

int batch_shared(bool fp16, const ChunkCall& t, const Prefixes& p, float* lse) {
    int rc = check_chunk(t);
    if (rc != QR_OK) return rc;
    if (p.count < 0 || p.count > 0x7fffffff || p.max_len < 0 || (p.count > 0 && t.window > 0) || (p.count > 1 && !p.members)) return QR_E_SHAPE;
    if (p.count > 0 && t.batch_size > 0 && (!p.indptr || !p.indices || !p.last_page_offset)) return QR_E_NULL;
    if (t.tokens == 0 || t.batch_size == 0) return rc;
    if (p.count > 0 && t.tokens * t.num_q_heads > 0xffffff0) return QR_E_SHAPE;            // (rows that one launch joins, 16 in 256 threads; their states are 142 GB)
    if ((uintptr_t)lse & 3) return QR_E_ALIGN;
    SharedPlan plan = shared_plan(fp16, t, p.count, p.max_len);
    const bool states = plan.parts > 1 || p.count > 0;
    if (states && (!t.workspace || ((uintptr_t)t.workspace & 15) || t.workspace_bytes < part_bytes(t.tokens, t.num_q_heads, plan.parts))) {
        if (p.count > 0) return QR_E_WORKSPACE;                // (the states are joined through memory)
        plan.own.splits = plan.parts = 1;
    }
    Chunk a = chunk_of(t);
    a.parts = plan.parts;
    a.lse = lse;
    hipStream_t st = (hipStream_t)t.stream;
    if (p.count > 0) {
        Chunk b = a;
        b.c.indptr = (const int32_t*)p.indptr, b.c.indices = (const int32_t*)p.indices, b.c.last_page_offset = (const int32_t*)p.last_page_offset;
        b.c.batch_size = (int)p.count;
        b.members = (const int32_t*)p.members;
        b.prefix = 1, b.per_place = kNoPlace;
        b.states = 1;
        b.part_at = plan.joined ? 0 : plan.own.splits;
        rc = plan.paired ? launch_pair(fp16, plan, b, a, st) : launch_chunk<true>(fp16, plan.prefix, b, st);
        if (rc != QR_OK) return rc;
        if (plan.joined) a.parts = 1, a.join = plan.parts, a.members = b.members, a.prefixes = (int)p.count;
    }
    a.states = a.parts > 1;
    if (!plan.paired) rc = launch_chunk<true>(fp16, plan.own, a, st);
    if (rc != QR_OK || a.parts == 1) return rc;
    Joined j;
    j.part = a.part, j.starts = a.starts, j.members = (const int32_t*)p.members;
    j.o = a.o, j.lse = lse, j.o_stride = t.o_stride;
    j.batch = (int)t.batch_size, j.tokens = (int)t.tokens, j.heads = t.num_q_heads, j.prefixes = (int)p.count, j.own = plan.own.splits, j.parts = plan.parts;
    j.per_head = divisor_of(t.num_q_heads);
    const int64_t rows = t.tokens * t.num_q_heads;
    if (rows <= 32 * (int64_t)qr_device().cus) chunk_join_kernel<4><<<dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st>>>(j);
    else chunk_join_kernel<1><<<dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st>>>(j);
    return qr_launch_status();
}

}  // namespace

extern "C" size_t qr_batch_chunk_workspace_bytes(int fp16_pages, int64_t tokens, int num_q_heads, int num_heads, int64_t batch_size, int64_t max_new_len,
                                                 int64_t max_seq_len, int64_t window, int64_t sinks) {
    if (tokens <= 0 || num_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_heads || batch_size <= 0 || batch_size > 0x7fffffff) return 0;
    if (tokens > 0x3fffffff || tokens * num_q_heads > 0x3fffffff || num_q_heads / num_heads > 1024 || num_heads > kMostHeads) return 0;        // (the call itself refuses them)
    const int splits = chunk_plan(fp16_pages != 0, tokens, num_q_heads / num_heads, num_heads, batch_size, max_new_len, max_seq_len, window, sinks).splits;
    return chunk_part_bytes(tokens, num_q_heads, splits);
}

#define QR_CHUNK_ENTRY(NAME, FP16)                                                                                                                \
    extern "C" int NAME(void* o, int64_t o_stride, const void* q, int64_t q_stride, int q_had_mode, const void* seqlen_indptr_or_null,            \
                        int64_t tokens, int num_q_heads, const void* kv_data, const void* kv_param, const void* kv_indptr,                         \
                        const void* kv_indices, const void* last_page_offset, int64_t num_pages, int num_layers, int layer_idx, int num_heads,     \
                        int page_size, int head_dim, int64_t batch_size, int64_t max_new_len, int64_t max_seq_len, int64_t window, int64_t sinks,  \
                        void* workspace, size_t workspace_bytes, void* stream) {                                                                  \
        return batch_chunk(FP16, ChunkCall{o, o_stride, q, q_stride, q_had_mode, seqlen_indptr_or_null, tokens, num_q_heads, kv_data, kv_param,     \
                                           kv_indptr, kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads, page_size,       \
                                           head_dim, batch_size, max_new_len, max_seq_len, window, sinks, workspace, workspace_bytes, stream});    \
    }
QR_CHUNK_ENTRY(qr_batch_chunk_i4, false)
QR_CHUNK_ENTRY(qr_batch_chunk_f16, true)

extern "C" size_t qr_batch_shared_workspace_bytes(int fp16_pages, int64_t tokens, int num_q_heads, int num_heads, int64_t batch_size, int64_t max_new_len,
                                                  int64_t max_seq_len, int64_t window, int64_t sinks, int64_t prefixes, int64_t max_prefix_len) {
    if (tokens <= 0 || num_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_heads || batch_size <= 0 || batch_size > 0x7fffffff || prefixes < 0 || prefixes > 0x7fffffff) return 0;
    if (tokens > 0x3fffffff || tokens * num_q_heads > 0x3fffffff || num_q_heads / num_heads > 1024 || num_heads > kMostHeads) return 0;        // (the call itself refuses them)
    ChunkCall t{};
    t.starts = &t;                     // (the caller gives max_new_len 1 where there are no bounds)
    t.tokens = tokens, t.num_q_heads = num_q_heads, t.num_heads = num_heads, t.batch_size = batch_size;
    t.max_new_len = max_new_len, t.max_seq_len = max_seq_len, t.window = window, t.sinks = sinks;
    const int parts = shared_plan(fp16_pages != 0, t, prefixes, max_prefix_len).parts;
    return prefixes > 0 ? part_bytes(tokens, num_q_heads, parts) : chunk_part_bytes(tokens, num_q_heads, parts);
}

#define QR_SHARED_ENTRY(NAME, FP16)                                                                                                                   \
    extern "C" int NAME(void* o, int64_t o_stride, void* lse_or_null, const void* q, int64_t q_stride, int q_had_mode,                                 \
                        const void* seqlen_indptr_or_null, int64_t tokens, int num_q_heads, const void* kv_data, const void* kv_param,                \
                        const void* kv_indptr, const void* kv_indices, const void* last_page_offset, int64_t num_pages, int num_layers,               \
                        int layer_idx, int num_heads, int page_size, int head_dim, int64_t batch_size, int64_t max_new_len, int64_t max_seq_len,      \
                        int64_t window, int64_t sinks, const void* prefix_indptr, const void* prefix_indices, const void* prefix_last_page_offset,    \
                        const void* prefix_sequences_or_null, int64_t prefixes, int64_t max_prefix_len, void* workspace, size_t workspace_bytes,      \
                        void* stream) {                                                                                                               \
        return batch_shared(FP16, ChunkCall{o, o_stride, q, q_stride, q_had_mode, seqlen_indptr_or_null, tokens, num_q_heads, kv_data, kv_param,       \
                                            kv_indptr, kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads, page_size,          \
                                            head_dim, batch_size, max_new_len, max_seq_len, window, sinks, workspace, workspace_bytes, stream},       \
                            Prefixes{prefix_indptr, prefix_indices, prefix_last_page_offset, prefix_sequences_or_null, prefixes, max_prefix_len},     \
                            (float*)lse_or_null);                                                                                                     \
    }
QR_SHARED_ENTRY(qr_batch_shared_i4, false)
QR_SHARED_ENTRY(qr_batch_shared_f16, true)
