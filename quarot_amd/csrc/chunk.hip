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

// ALIGNED: pages of a multiple of 16 positions, so that each half of a step lies in one page.
template <int NB, int NW, bool F16, bool ALIGNED>
__global__ __launch_bounds__(64 * NW, NB == 2 || F16 ? 2 : 3) void chunk_rows_kernel(Chunk a, Divisor pages) {
    extern __shared__ __attribute__((aligned(16))) f32x4 st4[];            // per wave and row: maximum, sum, -, -, 128 outputs
    const PagedKV& c = a.c;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int id = divided(blockIdx.x, a.per_split), split = blockIdx.x - id * a.splits, item = divided(id, a.per_head), h = id - item * c.num_heads;
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

    for (int tile = first_tile; tile * 16 * NB < rows; tile += a.tiles) {
        const int r0 = tile * 16 * NB, r1 = r0 + 16 * NB < rows ? r0 + 16 * NB : rows;
        const int lowest = first_place + divided(r0, a.per_group), highest = first_place + divided(r1 - 1, a.per_group);
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
            place[nb] = in ? first_place + t : -1;
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
                if (a.splits == 1) {
                    const float inv = D == 0.f ? 0.f : 1.f / D;                 // (a row that sees nothing is zero)
                    u32x2* const dst = (u32x2*)(a.o + (int64_t)(start + t) * a.o_stride + (int64_t)head * 128) + PER * l;
#pragma unroll
                    for (int i = 0; i < PER; ++i) dst[i] = u32x2{cvt_f16x2(O[i][0] * inv, O[i][1] * inv), cvt_f16x2(O[i][2] * inv, O[i][3] * inv)};
                } else {
                    float* dst = a.part + (((int64_t)(start + t) * (c.num_heads * a.group) + head) * a.splits + split) * 132;
                    if (l == 0) dst[0] = M, dst[1] = D;
#pragma unroll
                    for (int i = 0; i < PER; ++i) *((f32x4*)dst + 1 + PER * l + i) = O[i];
                }
            }
        }
    }
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
    int nb, nw, tiles, splits;
};
constexpr size_t kMostParts = (size_t)1 << 30;
constexpr int kMostHeads = 65536;                          // (with most splits a sequence's heads are a launch)
size_t chunk_part_bytes(int64_t tokens, int64_t q_heads, int splits) { return splits > 1 ? (size_t)tokens * q_heads * splits * 132 * sizeof(float) : 0; }
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

template <bool F16, bool ALIGNED>
int launch_rows(const ChunkPlan& plan, const Chunk& a, Divisor pages, int64_t groups, hipStream_t st) {
    using Kernel = void (*)(Chunk, Divisor);
    const Kernel kernel = plan.nb == 2 ? (plan.nw == 8 ? chunk_rows_kernel<2, 8, F16, ALIGNED> : chunk_rows_kernel<2, 4, F16, ALIGNED>)
                                       : (F16 || plan.nw == 4 ? chunk_rows_kernel<1, 4, F16, ALIGNED> : chunk_rows_kernel<1, F16 ? 4 : 12, F16, ALIGNED>);
    const size_t lds = (size_t)plan.nw * 16 * 33 * sizeof(f32x4);
    const hipError_t e = qr_allow_dynamic_lds((const void*)kernel, lds);
    if (e != hipSuccess) return (int)e;
    kernel<<<dim3((unsigned)groups), dim3(64 * plan.nw), lds, st>>>(a, pages);
    return qr_launch_status();
}

int batch_chunk(bool fp16, void* o, int64_t o_stride, const void* q, int64_t q_stride, int q_had_mode, const void* seqlen_indptr_or_null, int64_t tokens,
                int num_q_heads, const void* kv_data, const void* kv_param, const void* kv_indptr, const void* kv_indices, const void* last_page_offset,
                int64_t num_pages, int num_layers, int layer_idx, int num_heads, int page_size, int head_dim, int64_t batch_size, int64_t max_new_len,
                int64_t max_seq_len, int64_t window, int64_t sinks, void* workspace, size_t workspace_bytes, void* stream) {
    const int rc = qr_internal_check_paged_cache(kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads,
                                                 page_size, head_dim, batch_size);
    if (rc != QR_OK) return rc;
    if (q_had_mode != 0 && q_had_mode != 1) return QR_E_DTYPE;
    if (tokens < 0 || num_q_heads <= 0 || num_q_heads % num_heads || window < 0 || sinks < 0 || max_new_len < 0 || max_seq_len < 0) return QR_E_SHAPE;
    if (tokens == 0 || batch_size == 0) return QR_OK;
    if (!seqlen_indptr_or_null && tokens != batch_size) return QR_E_SHAPE;       // one new token per sequence
    if (!o || !q) return QR_E_NULL;
    if (((uintptr_t)q & 15) || ((uintptr_t)o & 15) || q_stride % 8 || o_stride % 8) return QR_E_ALIGN;
    const int64_t width = (int64_t)num_q_heads * 128;
    if (q_stride < width || o_stride < width || tokens > 0x3fffffff || tokens * num_q_heads > 0x3fffffff || num_q_heads / num_heads > 1024 || num_heads > kMostHeads)
        return QR_E_SHAPE;
    const ChunkPlan plan = chunk_plan(fp16, tokens, num_q_heads / num_heads, num_heads, batch_size, seqlen_indptr_or_null ? max_new_len : 1, max_seq_len, window, sinks);
    Chunk a;
    a.c = qr_internal_paged_kv((void*)kv_data, (void*)kv_param, kv_indptr, kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads,
                               page_size, batch_size);
    a.q = (const f16*)q;
    a.o = (f16*)o;
    a.starts = (const int32_t*)seqlen_indptr_or_null;
    a.q_stride = q_stride, a.o_stride = o_stride;
    a.tokens = (int)tokens;
    a.group = num_q_heads / num_heads;
    a.per_group = divisor_of(a.group);
    a.per_head = divisor_of(num_heads);
    a.tiles = plan.tiles;
    a.window = (int)(window > 0x3fffffff ? 0 : window);    // (longer than any sequence)
    a.sinks = (int)(sinks > 0x3fffffff ? 0x3fffffff : sinks);
    a.q_had = q_had_mode;
    a.splits = plan.splits;
    if (a.splits > 1 && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < chunk_part_bytes(tokens, num_q_heads, a.splits))) a.splits = 1;
    a.per_split = divisor_of(a.splits);
    a.part = (float*)workspace;
    // A launch has fewer than 2^32 threads: fewer tiles at a time where hints are missing (a workgroup goes on to the next one behind them), then fewer sequences
    const int64_t most = 0xffffffffll / (plan.nb == 0 ? 256 : 64 * plan.nw), wide = (int64_t)num_heads * a.splits;
    if (batch_size * wide * plan.tiles > most) a.tiles = (int)(batch_size * wide < most ? most / (batch_size * wide) : 1);
    const int64_t at_once = batch_size * wide <= most ? batch_size : most / wide;
    hipStream_t st = (hipStream_t)stream;
    const Divisor pages = divisor_of(page_size);
    const bool aligned = page_size % 16 == 0;
    int lrc = QR_OK;
    for (int64_t first = 0; first < batch_size && lrc == QR_OK; first += at_once) {
        Chunk some = a;
        some.c.batch_size = (int)(batch_size - first < at_once ? batch_size - first : at_once);
        some.c.indptr += first, some.c.last_page_offset += first;
        if (a.starts) some.starts += first;
        else some.q += first * q_stride, some.o += first * o_stride, some.part += a.splits > 1 ? first * num_q_heads * a.splits * 132 : 0;
        const int64_t groups = some.c.batch_size * wide * a.tiles;
        lrc = plan.nb == 0 ? qr_internal_chunk_tiles(fp16, some, pages, groups, st)
              : fp16       ? (aligned ? launch_rows<true, true>(plan, some, pages, groups, st) : launch_rows<true, false>(plan, some, pages, groups, st))
                           : (aligned ? launch_rows<false, true>(plan, some, pages, groups, st) : launch_rows<false, false>(plan, some, pages, groups, st));
    }
    if (lrc != QR_OK || a.splits == 1) return lrc;
    chunk_merge_kernel<<<dim3((unsigned)((tokens * num_q_heads + 3) / 4)), dim3(64), 0, st>>>(a.part, a.starts, (int)batch_size, (int)tokens, num_q_heads, divisor_of(num_q_heads),
                                                                                              a.splits, a.o, o_stride);
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
        return batch_chunk(FP16, o, o_stride, q, q_stride, q_had_mode, seqlen_indptr_or_null, tokens, num_q_heads, kv_data, kv_param, kv_indptr,    \
                           kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads, page_size, head_dim, batch_size,           \
                           max_new_len, max_seq_len, window, sinks, workspace, workspace_bytes, stream);                                          \
    }
QR_CHUNK_ENTRY(qr_batch_chunk_i4, false)
QR_CHUNK_ENTRY(qr_batch_chunk_f16, true)
