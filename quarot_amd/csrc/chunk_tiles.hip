// Attention of new tokens over the paged cache for many rows of a (sequence, key head): the mathematics of chunk.hip on tiles of 256 rows.
//
// Eight waves share the cached vectors of a step of 64 positions: each is unpacked once per workgroup, from registers into LDS, as the fp16
// operand that the matrix instructions take.  A wave holds 32 rows, the positions in its registers (chunk.hip: no exchange between lanes from
// the first product to the second), and of the second product's operand 132 rows: the 128 dimensions, and the reciprocal 1 / f_j and the zero
// point zero_j / f_j of every position as pairs of fp16 numbers (22 bits of each).  Their sums are those of the weights as they were
// rounded, sum p_j and sum p_j zero_j with p_j = fp16(weight_j f_j) / f_j, so a rounding changes a weight and nothing else.
#include "qr_chunk.h"

namespace {

constexpr int kRows = 256, kStep = 64;
// a step's place in LDS
constexpr int kKeys = 0, kValues = 16384, kValueRows = 133, kSlope = kValues + kValueRows * 128, kOffset = kSlope + 256, kFactor = kOffset + 256,
              kThere = kFactor + 128, kBuffer = (kThere + 8 + 255) / 256 * 256;

// n / d for n below 2^30: umulhi(4 n, inverse) >> shift
struct Divisor {
    u32 inverse, shift;
};
__device__ __forceinline__ int divided(int n, Divisor d) { return (int)(__umulhi((u32)n << 2, d.inverse) >> d.shift); }

// What a thread has fetched of a step: two of the sixteen pieces of a key and the parameters of that position, and four positions' values in four
// dimensions.
template <bool F16>
struct Codes {
    u32x4 k4[F16 ? 2 : 1];
    u32x2 k2;
    u32x2 v2[F16 ? 4 : 1];
    unsigned short v1[F16 ? 1 : 4];
    u32 kp, vp;                        // of the key's position
    u32 scales[4];                     // of the four positions ({scale, zero})
    bool k_there;
    u32 v_there;                       // bit i: position i of the four
};

// weight times factor -> fp16, rounded once: two weights, two factors (a pair of fp16 numbers)
__device__ __forceinline__ u32 scaled_pair(float w0, float w1, u32 factors) {
    u32 r;
    asm("v_fma_mixlo_f16 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "=v"(r) : "v"(w0), "v"(factors));
    asm("v_fma_mixhi_f16 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "+v"(r) : "v"(w1), "v"(factors));
    return r;
}

// ALIGNED: pages of a multiple of 16 positions, so that a wave's eight keys and its sixteen positions of values lie in one page each
template <bool F16, bool ALIGNED>
__global__ __launch_bounds__(512, 2) void chunk_tiles_kernel(Chunk a, Divisor pages) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const PagedKV& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;
    int id = blockIdx.x;
    const int split = id % a.splits;
    id /= a.splits;
    const int kvh_all = c.num_heads;
    const int pair = id % (kvh_all * c.batch_size);        // (sequence, key head): neighbours are on different XCDs, a pair's tiles on one where 8 divides their number
    const int tile = a.tiles - 1 - id / (kvh_all * c.batch_size);                  // the tiles with most positions first
    const int b = pair / kvh_all, head = pair - b * kvh_all;
    const Fresh tokens = fresh_of(a, b);
    const int rows = tokens.count * a.group;
    const int p0 = c.indptr[b], npages = c.indptr[b + 1] - p0;
    const int len = npages > 0 ? (npages - 1) * c.page_size + c.last_page_offset[b] : 0;
    const int64_t page_slots = (int64_t)c.num_layers * 2 * c.num_heads * c.page_size;
    const int64_t head_slots = ((int64_t)c.layer_idx * 2 * c.num_heads + head) * c.page_size;
    const int64_t kv_slots = (int64_t)c.num_heads * c.page_size;

    // rows of the operand that never change: fp16 pages have the weights' sum by a row of ones, and none are read beyond
    for (int i = tid; i < 2 * 5 * 32; i += 512) {
        const int at = i % 160, row = at >> 5;
        *(u32*)(lds + (i / 160) * kBuffer + kValues + (128 + row) * 128 + (at & 31) * 4) = F16 && row == 0 ? 0x3C003C00u : 0u;
    }

    for (int r_tile = tile * kRows; r_tile < rows; r_tile += a.tiles * kRows) {
        const int r_end = r_tile + kRows < rows ? r_tile + kRows : rows;
        const Steps steps = steps_of<6>(a, len - tokens.count + r_tile / a.group, len - tokens.count + (r_end - 1) / a.group);
        const int s_begin = (int)((int64_t)steps.all * split / a.splits), s_end = (int)((int64_t)steps.all * (split + 1) / a.splits);
        // the wave's rows
        const int r0 = r_tile + 32 * wave, r = r0 + n;
        const bool in = r < rows;
        const int t = (in ? r : r_tile) / a.group, q_head = head * a.group + (in ? r : r_tile) - t * a.group;
        const int place = in ? len - tokens.count + t : -1;
        const int r_last = r0 + 31 < rows ? r0 + 31 : rows - 1;
        const int lowest = r0 < rows ? len - tokens.count + r0 / a.group : -1, highest = r0 < rows ? len - tokens.count + r_last / a.group : -1;

        // the queries: lane (n, h) holds dimensions 16 s + 8 h .. + 7 of row n
        u32x4 qf[8];
        float qsum;
        {
            const u32x4* src = (const u32x4*)(a.q + (int64_t)(tokens.start + t) * a.q_stride + (int64_t)q_head * 128) + h;
#pragma unroll
            for (int s = 0; s < 8; ++s) qf[s] = in ? src[2 * s] : u32x4{0, 0, 0, 0};
            if (a.q_had) {
                float v[64];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const f16x2 p = as_f16x2(qf[i >> 2][i & 3]);
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
                    v[i] = h ? as_f32(e.x) - as_f32(e.y) : as_f32(e.x) + as_f32(e.y);
                }
#pragma unroll
                for (int i = 0; i < 32; ++i) qf[i >> 2][i & 3] = narrow_f16x2(v[2 * i] * kScale, v[2 * i + 1] * kScale);
            }
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const f16x2 p = as_f16x2(qf[i >> 2][i & 3]);
                sum += (float)p[0] + (float)p[1];
            }
            const u32x2 e = both_halves<32>(as_u32(sum));
            qsum = as_f32(e.x) + as_f32(e.y);
            if (!F16) {
#pragma unroll
                for (int s = 0; s < 8; ++s) qf[s] = query_for_codes(qf[s]);
            }
        }

        // ---- a step's way into LDS.  Thread (key, e) takes pieces 2 e, 2 e + 1 of a key; thread (four keys, word, half) four keys' values in dimensions
        // 8 word + 4 half ..  The four keys are 32 kb + 16 tt + 8 jj + 4 hh ..: what lane half hh of the second product takes in step tt as its
        // jj-th half.
        const int key = tid >> 3, e = tid & 7;
        const int jj = tid & 1, half = tid >> 1 & 1, word = tid >> 2 & 15, piece = tid >> 6;           // piece: 4 kb + 2 tt + hh
        const int four = 32 * (piece >> 2) + 16 * (piece >> 1 & 1) + 8 * jj + 4 * (piece & 1);
        const int v_row = 32 * (2 * (word & 1) + half) + 8 * (word >> 2) + 4 * (word >> 1 & 1);
        auto slot_at = [&](int pos, bool& there) {
            const int it = divided(pos, pages);
            const u32 entry = (u32)(pos - it * c.page_size);
            const bool inside = pos < len && it < npages && entry < (u32)c.page_size;
            const int page = npages > 0 ? c.indices[p0 + (inside ? it : 0)] : -1;
            there = inside && page >= 0 && page < c.num_pages;
            return there ? page * page_slots + head_slots + entry : head_slots;
        };
        auto fetch = [&](Codes<F16>& f, int s) {
            const int at = steps.at(s) * kStep;
            // (a position that is not there reads the first ones of page 0)
            if (ALIGNED) {
                bool k_page, v_page;
                const int v_at = at + 32 * (wave >> 2) + 16 * (wave >> 1 & 1);              // (piece is the wave's number)
                const int64_t kb = slot_at(at + 8 * wave, k_page), vb = slot_at(v_at, v_page) + kv_slots;
                const uint32_t k_lane = lane >> 3, v_lane = 8 * jj + 4 * (wave & 1);
                f.k_there = k_page && at + key < len;
                f.v_there = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) f.v_there |= (v_page && v_at + (int)v_lane + i < len ? 1u : 0u) << i;
                const uint8_t* const kd = c.data + kb * (F16 ? 256 : 64);
                const uint8_t* const vd = c.data + vb * (F16 ? 256 : 64);
                if (F16) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) f.k4[i] = *(const u32x4*)(kd + (k_lane * 256u + (uint32_t)e * 32u + 16u * i));
#pragma unroll
                    for (int i = 0; i < 4; ++i) f.v2[i] = *(const u32x2*)(vd + ((v_lane + i) * 256u + (uint32_t)(2 * word + half) * 8u));
                } else {
                    f.k2 = *(const u32x2*)(kd + (k_lane * 64u + (uint32_t)e * 8u));
                    const uint8_t* const kp = (const uint8_t*)(c.param + kb);
                    f.kp = *(const u32*)(kp + k_lane * 4u);
                    f.vp = *(const u32*)((const uint8_t*)(c.param + kb + kv_slots) + k_lane * 4u);
                    const uint8_t* const vp = (const uint8_t*)(c.param + vb);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        f.v1[i] = *(const unsigned short*)(vd + ((v_lane + i) * 64u + (uint32_t)(2 * word + half) * 2u));
                        f.scales[i] = *(const u32*)(vp + (v_lane + i) * 4u);
                    }
                }
            } else {
                const int64_t ks = slot_at(at + key, f.k_there);
                if (F16) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) f.k4[i] = ((const u32x4*)c.data)[ks * 16 + 2 * e + i];
                } else {
                    f.k2 = ((const u32x2*)c.data)[ks * 8 + e];
                    f.kp = c.param[ks], f.vp = c.param[ks + kv_slots];
                }
                f.v_there = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    bool there;
                    const int64_t vs = slot_at(at + four + i, there) + kv_slots;
                    f.v_there |= (there ? 1u : 0u) << i;
                    if (F16) {
                        f.v2[i] = ((const u32x2*)c.data)[vs * 32 + 2 * word + half];
                    } else {
                        f.v1[i] = ((const unsigned short*)c.data)[vs * 32 + 2 * word + half];
                        f.scales[i] = c.param[vs];
                    }
                }
            }
        };
        auto place_codes = [&](const Codes<F16>& f, uint8_t* buf) {
            // the key: piece p of 16 at p ^ (key % 16)
            u32x4* const krow = (u32x4*)(buf + kKeys + key * 256);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                krow[(2 * e + i) ^ (key & 15)] = F16 ? f.k4[i] : codes_of(f.k2[i]);
            }
            const int k_at = (key >> 5) * 32 + (key >> 4 & 1) * 16 + (key >> 2 & 1) * 8 + (key >> 3 & 1) * 4 + (key & 3);       // its place in the order of the second product
            if (!F16) {
                const f16x2 p = as_f16x2(f.kp), v = as_f16x2(f.k_there ? f.vp : kNoParameters);
                const float factor = factor_of((float)v[0], power_of((float)v[0])), recip = __builtin_amdgcn_rcpf(factor), zero = (float)v[1] * recip;
                const f16 recip_hi = (f16)recip, zero_hi = (f16)zero;
                if (e == 0) {
                    ((float*)(buf + kSlope))[k_at] = (float)p[0] * (kLog2e * kScale * kCodeUnit);
                    ((float*)(buf + kOffset))[k_at] = (float)p[1] * -(kLog2e * kScale);
                    ((f16*)(buf + kFactor))[k_at] = (f16)factor;
                    f16* const extra_rows = (f16*)(buf + kValues + 128 * 128) + k_at;
                    extra_rows[0] = recip_hi, extra_rows[64] = (f16)(recip - (float)recip_hi);
                    extra_rows[128] = zero_hi, extra_rows[192] = (f16)(zero - (float)zero_hi);
                }
            }
            {
                const uint64_t there = __builtin_amdgcn_ballot_w64(f.k_there);
                if (lane == 0) {
                    uint32_t bits = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) bits |= (uint32_t)(there >> (8 * i) & 1) << i;
                    buf[kThere + wave] = (uint8_t)bits;
                }
            }
            // the values: row v_row + i holds dimension 8 word + 4 half + i
            uint8_t* const vrow = buf + kValues + v_row * 128 + jj * 8;
            u32 out[4][2];
            if (F16) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    u32x2 x = f.v2[2 * k], y = f.v2[2 * k + 1];
                    if (!(f.v_there >> (2 * k) & 1)) x = u32x2{0, 0};
                    if (!(f.v_there >> (2 * k + 1) & 1)) y = u32x2{0, 0};
                    out[0][k] = __builtin_amdgcn_perm(y.x, x.x, 0x05040100u);
                    out[1][k] = __builtin_amdgcn_perm(y.x, x.x, 0x07060302u);
                    out[2][k] = __builtin_amdgcn_perm(y.y, x.y, 0x05040100u);
                    out[3][k] = __builtin_amdgcn_perm(y.y, x.y, 0x07060302u);
                }
            } else {
                u32 vp[4], power[2];
#pragma unroll
                for (int i = 0; i < 4; ++i) vp[i] = (f.v_there >> i & 1) ? f.scales[i] : kNoParameters;
                bool plain = true;
#pragma unroll
                for (int k = 0; k < 2; ++k) power[k] = powers_of(vp[2 * k], vp[2 * k + 1], plain);
                const u32 w[2] = {(u32)f.v1[0] | (u32)f.v1[1] << 16, (u32)f.v1[2] | (u32)f.v1[3] << 16};
                if (__builtin_amdgcn_ballot_w64(!plain) == 0) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const u32x4 scaled = scaled_codes(w[k], power[k]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) out[i][k] = scaled[i];
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const u32x4 scaled = scaled_codes_slow(w[k], vp[2 * k], vp[2 * k + 1]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) out[i][k] = scaled[i];
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = v_row + i;
                *(u32x2*)(vrow + i * 128 + ((piece ^ (row >> 1 & 7) ^ (row >> 5 & 1)) << 4)) = u32x2{out[i][0], out[i][1]};
            }
        };

        f32x16 acc[4], extra;
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[0][i] = acc[1][i] = acc[2][i] = acc[3][i] = extra[i] = 0.f;
        float m = 0.f, limit = -3e38f;                     // (until the row has seen a position, any logit moves its maximum)

        auto consume = [&](const uint8_t* buf, int s) {
            const int at = steps.at(s) * kStep;
            if (at > highest) return;                      // (nothing in it for this wave's rows)
            const uint64_t there = *(const uint64_t*)(buf + kThere);
            const bool whole = at + kStep - 1 <= lowest && (a.window == 0 || at > highest - a.window || at + kStep - 1 < a.sinks) && ~there == 0;
            f32x16 x[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) x[0][i] = x[1][i] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const u32x4 k = ((const u32x4*)(buf + kKeys + (32 * kb + n) * 256))[(2 * i + h) ^ (n & 15)];
                    x[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, qf[i]), x[kb], 0, 0, 0);
                }
            // logits less the running maximum, base 2; register 8 tt + j of half h is place 32 kb + 16 tt + 8 h + j of the second product's order
            float top = -__builtin_inff();
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const f32x4* slope = (const f32x4*)(buf + kSlope) + 8 * kb + 4 * tt + 2 * h;
                    const f32x4* offset = (const f32x4*)(buf + kOffset) + 8 * kb + 4 * tt + 2 * h;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (F16) x[kb][8 * tt + j] = __builtin_fmaf(x[kb][8 * tt + j], kLog2e * kScale, -m);
                        else x[kb][8 * tt + j] = __builtin_fmaf(x[kb][8 * tt + j], slope[j >> 2][j & 3], __builtin_fmaf(offset[j >> 2][j & 3], qsum, -m));
                    }
                }
            if (!whole) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int k = 32 * kb + 8 * (i >> 2) + 4 * h + (i & 3), pos = at + k;
                        const bool sees = pos <= place && (a.window == 0 || pos > place - a.window || pos < a.sinks) && (there >> k & 1);
                        x[kb][i] = sees ? x[kb][i] : -__builtin_inff();
                    }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, __builtin_fmaxf(x[0][i], x[1][i]));
            if (__builtin_amdgcn_ballot_w64(top > limit)) {
                const u32x2 both = both_halves<32>(as_u32(top));
                top = __builtin_fmaxf(as_f32(both.x), as_f32(both.y));
                const bool moves = top > (limit < 0.f ? limit : 0.f);
                const float by = moves ? top : 0.f, keep = __builtin_amdgcn_exp2f(-by);
                limit = moves ? kGrow : limit;
                m += by;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    x[0][i] -= by, x[1][i] -= by;
                    acc[0][i] *= keep, acc[1][i] *= keep, acc[2][i] *= keep, acc[3][i] *= keep, extra[i] *= keep;
                }
            }
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const int piece_at = 4 * kb + 2 * tt + h;
                    u32x4 packed;
                    const u32x4 factor = F16 ? u32x4{} : *(const u32x4*)(buf + kFactor + piece_at * 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float w0 = __builtin_amdgcn_exp2f(x[kb][8 * tt + 2 * j]), w1 = __builtin_amdgcn_exp2f(x[kb][8 * tt + 2 * j + 1]);
                        packed[j] = F16 ? cvt_f16x2(w0, w1) : scaled_pair(w0, w1, factor[j]);
                    }
                    const f16x8 p = __builtin_bit_cast(f16x8, packed);
#pragma unroll
                    for (int db = 0; db < 4; ++db) {
                        const u32x4 v = ((const u32x4*)(buf + kValues + (32 * db + n) * 128))[piece_at ^ (n >> 1 & 7) ^ (db & 1)];
                        acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), p, acc[db], 0, 0, 0);
                    }
                    const u32x4 v = ((const u32x4*)(buf + kValues + (128 + (n < 4 ? n : 4)) * 128))[piece_at];
                    extra = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v), p, extra, 0, 0, 0);
                }
        };

        __syncthreads();                                   // (the rows above; the last tile's buffers)
        Codes<F16> f;
        if (s_begin < s_end) {
            fetch(f, s_begin);
            place_codes(f, lds);
            fetch(f, s_begin + 1 < s_end ? s_begin + 1 : s_begin);
        }
        __syncthreads();
        for (int s = s_begin; s < s_end; ++s) {
            uint8_t* const buf = lds + (s - s_begin & 1) * kBuffer;
            uint8_t* const other = lds + (s - s_begin + 1 & 1) * kBuffer;
            if (s + 1 < s_end) {
                place_codes(f, other);
                fetch(f, s + 2 < s_end ? s + 2 : s + 1);
            }
            consume(buf, s);
            __syncthreads();
        }

        // rows 0 .. 3 of the extra block, in the registers of the lower half: sums of weights (as pairs) and of weights times zero points
        float sum = F16 ? extra[0] : extra[0] + extra[1], zero = F16 ? 0.f : extra[2] + extra[3];
        sum = as_f32(both_halves<32>(as_u32(sum)).x);
        if (!F16) zero = as_f32(both_halves<32>(as_u32(zero)).x);
        if (in) {
            // lane (n, h): dimensions 32 i + 16 h + 4 db + j of row n in register 4 i + j of block db
            if (a.splits == 1) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                u32x4* const dst = (u32x4*)(a.o + (int64_t)(tokens.start + t) * a.o_stride + (int64_t)q_head * 128) + 2 * h;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        u32x4 w;
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int db = 2 * k + (j >> 1), reg = 4 * i + 2 * (j & 1);
                            w[j] = cvt_f16x2((acc[db][reg] - zero) * inv, (acc[db][reg + 1] - zero) * inv);
                        }
                        dst[4 * i + k] = w;
                    }
            } else {
                float* const dst = a.part + (((int64_t)(tokens.start + t) * (c.num_heads * a.group) + q_head) * a.splits + split) * 132;
                if (h == 0) dst[0] = limit < 0.f ? kEmpty : m, dst[1] = sum;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int db = 0; db < 4; ++db)
                        *(f32x4*)(dst + 4 + 32 * i + 16 * h + 4 * db) = f32x4{acc[db][4 * i] - zero, acc[db][4 * i + 1] - zero, acc[db][4 * i + 2] - zero, acc[db][4 * i + 3] - zero};
            }
        }
    }
}

}  // namespace

int qr_internal_chunk_tiles(bool fp16, const Chunk& a, int64_t groups, hipStream_t st) {
    using Kernel = void (*)(Chunk, Divisor);
    const bool aligned = a.c.page_size % 16 == 0;
    const Kernel kernel = fp16 ? (aligned ? chunk_tiles_kernel<true, true> : chunk_tiles_kernel<true, false>)
                               : (aligned ? chunk_tiles_kernel<false, true> : chunk_tiles_kernel<false, false>);
    const hipError_t e = qr_allow_dynamic_lds((const void*)kernel, 2 * kBuffer);
    if (e != hipSuccess) return (int)e;
    const u32 log2 = a.c.page_size > 1 ? 64u - (u32)__builtin_clzll((unsigned long long)a.c.page_size - 1) : 0u;
    const Divisor pages{(u32)(((1ull << (30 + log2)) + (uint64_t)a.c.page_size - 1) / (uint64_t)a.c.page_size), log2};
    kernel<<<dim3((unsigned)groups), dim3(512), 2 * kBuffer, st>>>(a, pages);
    return qr_launch_status();
}
