// What attention gives to the cached positions, added up position by position, from the queries, the softmax's logarithmic sums and the keys:
//
//   W[b, h, j] += sum over the new tokens t of sequence b and the query heads g of key head h of exp( q[t, g] . k[j, h] / sqrt(128) - lse[t, g] )
//
// over the positions j that t sees (chunk.hip: all up to its own, or the last `window` and the first `sinks`).  A position belongs to one lane from
// its key to its sum: nothing is exchanged but the four partial sums of a column, no atomics, and the order of the additions is always the same.
//
// The logits are a product rows x positions, positions in the lanes: a position's scale and zero point are its lane's, sums over rows are sums of
// registers.  Int4 keys enter as codes, which fp16 holds exactly (chunk.hip); every q too: a code is shifted into its half's lowest four bits, so
// that no element of q is divided.  Logits, exponentials and sums are in 32 bits, nothing is rounded to fewer.
#include "qr_chunk.h"

namespace {

struct Weights {
    PagedKV c;
    const f16* q;
    const float* lse;
    float* sums;                      // [sequence, key head, capacity]
    const int32_t* starts;            // nullptr: one new token per sequence
    int64_t q_stride, capacity;
    int tokens, group, blocks, window, sinks, q_had;
    Divisor per_group, per_block, per_head;
};

__device__ __forceinline__ Fresh fresh_of(const Weights& a, int b) {
    if (!a.starts) return Fresh{b, 1, 1};
    int start = a.starts[b];
    const int end = a.starts[b + 1];
    start = start < 0 ? 0 : start;
    const int stop = end > a.tokens ? a.tokens : end;
    return Fresh{start, stop > start ? stop - start : 0, end > start ? end - start : 0};
}

// the codes of a word as in codes_of, all of them in a half's lowest four bits
__device__ __forceinline__ u32x4 low_codes_of(u32 w) {
    return u32x4{w & 0x000F000Fu, (w >> 4) & 0x000F000Fu, (w >> 8) & 0x000F000Fu, (w >> 12) & 0x000F000Fu};
}
// eight elements of q in the order of a word's codes: (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ u32x4 query_for_low_codes(u32x4 w) {
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
// A wave takes 64 positions of a (sequence, key head), lane by lane for their places, and all rows in tiles of 16: lane (n, g) holds quarter g of the
// keys of positions n, 16 + n, 32 + n and 48 + n.
constexpr int kWaves = 4;
template <bool F16>
__global__ __launch_bounds__(64 * kWaves) void weights_rows_kernel(Weights a, Divisor pages) {
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
    constexpr float kUnit = kLog2e * kScale * (F16 ? 1.f : kCodeUnit);

    const int highest = first_place + divided(rows - 1, a.per_group);
    auto sees = [&](int place, int pos) { return pos <= place && (a.window == 0 || pos > place - a.window || pos < a.sinks); };
    // blocks of 64 positions that some row sees
    struct {
        int near, far, all;
    } steps{0, 0, 0};
    if (highest >= 0) {
        const Steps s = [&] {
            Steps t{0, 0, 0};
            int from = 0;
            if (a.window > 0 && first_place - a.window + 1 > 0) {
                from = first_place - a.window + 1;
                const int sinks = a.sinks < from ? a.sinks : from;
                t.near = (sinks + 63) >> 6;
            }
            t.far = from >> 6;
            if (t.far < t.near) t.far = t.near;
            const int end = (highest >> 6) + 1;
            t.all = t.near + (end > t.far ? end - t.far : 0);
            return t;
        }();
        steps.near = s.near, steps.far = s.far, steps.all = s.all;
    }
    for (int block = first_block * kWaves + wave; block < steps.all; block += a.blocks * kWaves) {
        const int at = (block < steps.near ? block : block - steps.near + steps.far) * 64;
        // the lane's own position: where its key is
        const int pos = at + lane, it = divided(pos, pages);
        const u32 entry = (u32)(pos - it * c.page_size);
        const bool in = pos < len && it < npages && entry < (u32)c.page_size;
        const int page = c.indices[p0 + (in ? it : 0)];
        const bool there = in && page >= 0 && page < c.num_pages;
        const int64_t slot = there ? page * page_slots + head_slots + entry : head_slots;
        const u32 param = F16 ? 0u : c.param[slot];
        u32x4 k[4][4];
        float scale[4], zero[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const uint8_t* const kd = c.data + __shfl(slot, 16 * s + n, 64) * VEC + g * 16;
            if (F16) {
#pragma unroll
                for (int i = 0; i < 4; ++i) k[s][i] = *(const u32x4*)(kd + 64 * i);
            } else {
                const u32x4 w = *(const u32x4*)kd;
#pragma unroll
                for (int i = 0; i < 4; ++i) k[s][i] = low_codes_of(w[i]);
                const f16x2 p = as_f16x2((u32)__shfl((int)param, 16 * s + n, 64));
                scale[s] = (float)p[0] * kUnit, zero[s] = (float)p[1];
            }
        }
        // (sums of 16 tiles of rows, then of these: a long chain of additions would lose what is small)
        float sum[4] = {0.f, 0.f, 0.f, 0.f}, all_before[4] = {0.f, 0.f, 0.f, 0.f};
        for (int r0 = 0; r0 < rows; r0 += 16) {
            if ((r0 & 255) == 0) {
#pragma unroll
                for (int s = 0; s < 4; ++s) all_before[s] += sum[s], sum[s] = 0.f;
            }
            // queries: lane (n, g) holds dimensions 32 g + 8 i .. (fp16 pages: 32 i + 8 g ..) of row n
            const int r = r0 + n < rows ? r0 + n : r0, t = divided(r, a.per_group), head = h * a.group + r - t * a.group;
            const u32x4* src = (const u32x4*)(a.q + (int64_t)(mine.start + t) * a.q_stride + (int64_t)head * 128);
            u32x4 w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = src[F16 && !a.q_had ? 4 * i + g : 4 * g + i];
            float slope = 0.f;
            if (!F16) {
                if (a.q_had) hadamard_row(w, lane);
                float all = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const f16x2 p = as_f16x2(w[i >> 2][i & 3]);
                    all += (float)p[0] + (float)p[1];
                }
                slope = quarters_sum(all) * -(kLog2e * kScale);
            } else if (a.q_had) {
                hadamard_row(w, lane);
                // (dimensions 32 g + 8 i to 32 i + 8 g: lanes (n, 0..3) trade pieces)
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
            f32x4 x[4];
#pragma unroll
            for (int s = 0; s < 4; ++s) x[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f16x8 q = __builtin_bit_cast(f16x8, F16 ? w[i] : query_for_low_codes(w[i]));
#pragma unroll
                for (int s = 0; s < 4; ++s) x[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(q, __builtin_bit_cast(f16x8, k[s][i]), x[s], 0, 0, 0);
            }
            // register i of lane (n, g): row 4 g + i, position n
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = r0 + 4 * g + i, token = divided(row < rows ? row : 0, a.per_group), place = row < rows ? first_place + token : -1;
                const float lse = row < rows ? a.lse[(int64_t)(mine.start + token) * (c.num_heads * a.group) + h * a.group + row - token * a.group] : 0.f;
                const float less = lse * -kLog2e, mine_slope = F16 ? 0.f : __shfl(slope, 4 * g + i, 64);
                const bool any = lse != -__builtin_inff();         // (a row that has seen nothing gives nothing)
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const float y = F16 ? __builtin_fmaf(x[s][i], kUnit, less) : __builtin_fmaf(x[s][i], scale[s], __builtin_fmaf(zero[s], mine_slope, less));
                    sum[s] += any && sees(place, at + 16 * s + n) ? __builtin_amdgcn_exp2f(y) : 0.f;
                }
            }
        }
        float total = 0.f;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const float all = quarters_sum(sum[s] + all_before[s]);
            total = g == s ? all : total;
        }
        if (there && pos < a.capacity) {
            float* const to = a.sums + ((int64_t)b * c.num_heads + h) * a.capacity + pos;
            *to += total;
        }
    }
}

template <bool F16>
int launch_weights(const Weights& a, int64_t groups, hipStream_t st) {
    weights_rows_kernel<F16><<<dim3((unsigned)groups), dim3(64 * kWaves), 0, st>>>(a, divisor_of(a.c.page_size));
    return qr_launch_status();
}

int accumulate(bool fp16, void* weights, int64_t capacity, const void* q, int64_t q_stride, int q_had_mode, const void* lse, const void* starts, int64_t tokens,
               int num_q_heads, const void* kv_data, const void* kv_param, const void* kv_indptr, const void* kv_indices, const void* last_page_offset, int64_t num_pages,
               int num_layers, int layer_idx, int num_heads, int page_size, int head_dim, int64_t batch_size, int64_t max_new_len, int64_t max_seq_len, int64_t window,
               int64_t sinks, void* stream) {
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
    a.window = (int)(window > 0x3fffffff ? 0 : window);
    a.sinks = (int)(sinks > 0x3fffffff ? 0x3fffffff : sinks);
    a.q_had = q_had_mode;
    a.per_group = divisor_of(a.group), a.per_head = divisor_of(num_heads);
    // positions that the launch is sized for (what is longer is gone through in turns); a launch has fewer than 2^32 threads
    int64_t seen = max_seq_len > 0 && max_seq_len < capacity ? max_seq_len : capacity;
    const int64_t fresh = max_new_len > 0 && starts ? max_new_len : starts ? tokens : 1;
    if (a.window > 0 && a.sinks < seen && seen > a.window + fresh + a.sinks + 192) seen = a.window + fresh + a.sinks + 192;
    int64_t blocks = (seen + 64 * kWaves - 1) / (64 * kWaves);
    if (blocks > 0xffff) blocks = 0xffff;
    const int64_t most = 0xffffffffll / (64 * kWaves);
    if (batch_size * num_heads * blocks > most) blocks = batch_size * num_heads < most ? most / (batch_size * num_heads) : 1;
    a.blocks = (int)blocks, a.per_block = divisor_of(blocks);
    const int64_t wide = num_heads * blocks, at_once = batch_size * wide <= most ? batch_size : most / wide;
    int lrc = QR_OK;
    for (int64_t first = 0; first < batch_size && lrc == QR_OK; first += at_once) {
        Weights some = a;
        some.c.batch_size = (int)(batch_size - first < at_once ? batch_size - first : at_once);
        some.c.indptr += first, some.c.last_page_offset += first;
        some.sums += first * num_heads * capacity;
        if (a.starts) some.starts += first;
        else some.q += first * q_stride, some.lse += first * num_q_heads;
        lrc = fp16 ? launch_weights<true>(some, some.c.batch_size * wide, (hipStream_t)stream) : launch_weights<false>(some, some.c.batch_size * wide, (hipStream_t)stream);
    }
    return lrc;
}

}  // namespace

#define QR_WEIGHTS_ENTRY(NAME, FP16)                                                                                                                     \
    extern "C" int NAME(void* weights, int64_t capacity, const void* q, int64_t q_stride, int q_had_mode, const void* lse,                               \
                        const void* seqlen_indptr_or_null, int64_t tokens, int num_q_heads, const void* kv_data, const void* kv_param,                   \
                        const void* kv_indptr, const void* kv_indices, const void* last_page_offset, int64_t num_pages, int num_layers, int layer_idx,   \
                        int num_heads, int page_size, int head_dim, int64_t batch_size, int64_t max_new_len, int64_t max_seq_len, int64_t window,        \
                        int64_t sinks, void* stream) {                                                                                                   \
        return accumulate(FP16, weights, capacity, q, q_stride, q_had_mode, lse, seqlen_indptr_or_null, tokens, num_q_heads, kv_data, kv_param, kv_indptr, \
                          kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads, page_size, head_dim, batch_size, max_new_len,       \
                          max_seq_len, window, sinks, stream);                                                                                           \
    }
QR_WEIGHTS_ENTRY(qr_accumulate_weights_i4, false)
QR_WEIGHTS_ENTRY(qr_accumulate_weights_f16, true)
