// Eviction from the paged cache: which positions of a (sequence, key head) stay, and their move to the front.
#include "qr_chunk.h"

namespace {

// ---- which stay ------------------------------------------------------------------------------------------------------------------------------
// Of a sequence of more than `keep` positions the first `sinks`, the last `recent`, and of those between the ones of the largest sums, the lowest
// positions first among equal ones.  The least sum that stays is found digit by digit (11, 11 and 10 bits of the sums' order as integers) from
// histograms in LDS; then every wave goes through its own range of positions in order and writes those that stay behind what the waves before it have.
// One workgroup to a list, whose sums are read once, into registers: 32 lists of 2500 5.5 us, 256 lists of up to 16384 11.4, of which 4 are the launch; the rest is the chain of
// load, three histograms and the list, a barrier after each (sums read anew for every digit, one counter per bin: 24.8).  Two workgroups to a list would have to wait for each
// other.
struct Heavy {
    const float* sums;
    const int32_t* lengths;
    int32_t *kept, *left;
    int64_t capacity;
    int heads, keep, sinks, recent;
};
// sums in the order of unsigned integers: NaN below all numbers, both zeros the same
__device__ __forceinline__ u32 order_of(float v) {
    const u32 u = __builtin_bit_cast(u32, v);
    return v != v ? 0u : v == 0.f ? 0x80000000u : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
constexpr int kBins = 2048, kHeavyWaves = 16, kHeavyThreads = 64 * kHeavyWaves;

// running sums over a wave's lanes up to this one, and over each 16 of them
__device__ __forceinline__ int upto16(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);       // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
}
__device__ __forceinline__ int upto64(int v) {
    v = upto16(v);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);       // row_bcast 15, 31
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}
// of one number per wave: the sum of those of the waves before this one
__device__ __forceinline__ int of_waves_before(const int* counts, int lane, int wave) {
    const int v = counts[lane & 15];
    return __builtin_amdgcn_readlane(upto16(v) - v, wave);
}
__device__ __forceinline__ int lanes_before(uint64_t mask) { return __builtin_amdgcn_mbcnt_hi((u32)(mask >> 32), __builtin_amdgcn_mbcnt_lo((u32)mask, 0)); }

// HOLD > 0: a lane keeps its sums, at most that many, in registers; 0: they are read for every digit
// (They are left behind eight at a time where the list ends: to pass over the rest one by one cost 14 us instead of 7.8 at 4000 positions of a capacity of 32768, a branch at every
// one 12 - 20 % where all are there.)
template <int HOLD>
__global__ __launch_bounds__(kHeavyThreads) void heavy_positions_kernel(Heavy a) {
    // four counters per bin, a lane's by its number: half of a wave's sums have one of a few dozen leading digits, and would wait for each other
    __shared__ u32x4 bins[kBins];
    __shared__ u32 found[3];                               // the digit, how many lie above it, how many have it
    __shared__ int counts[3][kHeavyWaves], after[2][kHeavyWaves];
    const int b = blockIdx.x / a.heads, h = blockIdx.x - b * a.heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t held = a.lengths[b];
    const int len = (int)(held < 0 ? 0 : held > a.capacity ? a.capacity : held);
    if (h == 0 && tid == 0) a.left[b] = len < a.keep ? len : a.keep;
    int32_t* const kept = a.kept + (int64_t)blockIdx.x * a.keep;
    if (len <= a.keep) {
        for (int i = tid; i < a.keep; i += kHeavyThreads) kept[i] = i < len ? i : -1;
        return;
    }
    const int need = a.keep - a.sinks - a.recent, count = len - a.sinks - a.recent;          // 0 <= need < count
    const float* const sums = a.sums + (int64_t)blockIdx.x * a.capacity + a.sinks;
    const int each = ((count + kHeavyWaves - 1) / kHeavyWaves + 63) & ~63, from = wave * each, to = from + each < count ? from + each : count;
    // the wave's sums in the order of positions, 64 at a time
    u32 mine[HOLD > 0 ? HOLD : 1];
    if (HOLD > 0) {
        float v[HOLD > 0 ? HOLD : 1];
#pragma unroll
        for (int j = 0; j < HOLD; ++j) {
            if (j % 8 == 0 && from + 64 * j >= to) break;
            v[j] = from + 64 * j + lane < to ? sums[from + 64 * j + lane] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < HOLD; ++j) mine[j] = order_of(v[j]);
    }
    for (int i = tid; i < a.sinks; i += kHeavyThreads) kept[i] = i;
    for (int i = tid; i < a.recent; i += kHeavyThreads) kept[a.keep - a.recent + i] = len - a.recent + i;
    if (need == 0) return;
    auto go_through = [&](auto&& visit) {                  // visit(position, its sum's order, whether it is one); all lanes of a wave together
        if (HOLD > 0) {
#pragma unroll
            for (int j = 0; j < HOLD; ++j) {
                if (j % 8 == 0 && from + 64 * j >= to) break;
                visit(from + 64 * j + lane, mine[j], from + 64 * j + lane < to);         // (of a part of eight the others are none)
            }
        } else {
            for (int at = from; at < to; at += 64 * 8) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = at + 64 * j + lane < to ? sums[at + 64 * j + lane] : 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at + 64 * j < to) visit(at + 64 * j + lane, order_of(v[j]), at + 64 * j + lane < to);
            }
        }
    };

    u32 prefix = 0, above = 0;                             // the digits found so far; how many sums lie above all that have them
    int shift = 32;
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass < 2 ? 11 : 10, below = shift;
        shift -= bits;
        bins[tid] = bins[kHeavyThreads + tid] = u32x4{0, 0, 0, 0};
        __syncthreads();
        go_through([&](int, u32 k, bool is) {
            if (is && (pass == 0 || k >> (below & 31) == prefix)) atomicAdd((u32*)&bins[k >> shift & ((1u << bits) - 1)] + (lane & 3), 1u);
        });
        __syncthreads();
        // thread t has the bins 2 t and 2 t + 1 from the top; how many sums lie in the bins before its own
        const u32x4 c0 = bins[kBins - 1 - 2 * tid], c1 = bins[kBins - 2 - 2 * tid];
        const u32 b0 = c0[0] + c0[1] + c0[2] + c0[3], b1 = c1[0] + c1[1] + c1[2] + c1[3];
        const u32 upto = (u32)upto64((int)(b0 + b1));
        if (lane == 63) counts[pass][wave] = (int)upto;
        __syncthreads();
        const int waves_before = of_waves_before(counts[pass], lane, wave);
        const u32 before = above + (u32)waves_before + upto - b0 - b1, want = (u32)need;
        if (before < want && before + b0 >= want) found[0] = kBins - 1 - 2 * tid, found[1] = before, found[2] = b0;
        if (before + b0 < want && before + b0 + b1 >= want) found[0] = kBins - 2 - 2 * tid, found[1] = before + b0, found[2] = b1;
        __syncthreads();
        prefix = prefix << bits | found[0];
        above = found[1];
        if (above + found[2] == want) break;               // (all that share these digits stay)
    }
    const int equal = need - (int)above;                   // of those with these digits that many stay, the first ones
    if (HOLD > 0 && (u32)equal == found[2]) {
        // all of them: one comparison for each, kept in scalar registers between the count and the list
        uint64_t stay[HOLD > 0 ? HOLD : 1];
        int count_here = 0;
#pragma unroll
        for (int j = 0; j < HOLD; ++j) {
            if (j % 8 == 0 && from + 64 * j >= to) break;
            stay[j] = __builtin_amdgcn_ballot_w64(from + 64 * j + lane < to && mine[j] >> shift >= prefix);
            count_here += __popcll(stay[j]);
        }
        if (lane == 0) after[0][wave] = count_here;
        __syncthreads();
        int32_t* to_list = kept + a.sinks + of_waves_before(after[0], lane, wave);
#pragma unroll
        for (int j = 0; j < HOLD; ++j) {
            if (j % 8 == 0 && from + 64 * j >= to) break;
            if (stay[j] >> lane & 1) to_list[lanes_before(stay[j])] = a.sinks + from + 64 * j + lane;
            to_list += __popcll(stay[j]);
        }
        return;
    }
    int greater = 0, same = 0;
    go_through([&](int, u32 k, bool is) {
        greater += __popcll(__builtin_amdgcn_ballot_w64(is && k >> shift > prefix));
        same += __popcll(__builtin_amdgcn_ballot_w64(is && k >> shift == prefix));
    });
    if (lane == 0) after[0][wave] = greater, after[1][wave] = same;
    __syncthreads();
    // of the waves before this one: how many stay, how many have these digits
    int out = of_waves_before(after[0], lane, wave), seen = of_waves_before(after[1], lane, wave);
    out += seen < equal ? seen : equal;
    go_through([&](int i, u32 k, bool is) {
        k >>= shift;
        const uint64_t eq = __builtin_amdgcn_ballot_w64(is && k == prefix);
        const bool stays = is && (k > prefix || (k == prefix && seen + lanes_before(eq) < equal));
        const uint64_t all = __builtin_amdgcn_ballot_w64(stays);
        if (stays) kept[a.sinks + out + lanes_before(all)] = a.sinks + i;
        out += __popcll(all), seen += __popcll(eq);
    });
}

// ---- their move --------------------------------------------------------------------------------------------------------------------------------
// Entry i of the list of a (sequence, key head) goes to position i, in place.  The list ascends, so a position is never behind its entry's: a workgroup goes
// through one side's vectors (keys or values) in batches, all of a batch in registers before the first is written, and what it writes lies before every entry of
// the batches to come.
// Eight vectors' pieces a thread are under way at a time, page numbers and slots come from a list in LDS made for 2048 entries at once (looked up by every thread
// between its loads: 196 us where it takes 132).  1024 of 2048, 32 heads, int4: 7.0 us; fp16 pages, 32 x 2000 of up to 8001, 8 heads: 132 us, 4.1 TB/s read and written of a copy's
// 5.2: loads and stores take turns in a workgroup, three of which share a CU (two, with 94 registers for the next part of the list: 163).
struct Keep {
    PagedKV c;
    const int32_t* kept;
    float* sums;                       // [sequence, key head, capacity]; may be nullptr
    int64_t capacity;
    int keep, jobs;                    // workgroups per (sequence, key head): keys, values, sums
    Divisor pages;                     // of the page size
};
constexpr int kKeepThreads = 512, kListed = 2048;

template <bool F16>
__global__ __launch_bounds__(kKeepThreads, 4) void keep_positions_kernel(Keep a) {
    constexpr int LANES = F16 ? 16 : 4, EACH = kKeepThreads / LANES, TURNS = 8;              // lanes of a vector, vectors at a time
    __shared__ int64_t sources[kListed], targets[kListed];                                  // slots; a target of -1: nothing moves
    const PagedKV& c = a.c;
    const int id = blockIdx.x / a.jobs, side = blockIdx.x - id * a.jobs, b = id / c.num_heads, h = id - b * c.num_heads;
    const int tid = threadIdx.x, p0 = c.indptr[b], npages = c.indptr[b + 1] - p0;
    const int len = npages > 0 ? (npages - 1) * c.page_size + c.last_page_offset[b] : 0;
    const int32_t* const kept = a.kept + (int64_t)id * a.keep;
    if (side == 2) {
        float* const sums = a.sums + (int64_t)id * a.capacity;
        const int have = (int)(len < a.capacity ? len : a.capacity), end = a.keep < have ? a.keep : have;
        constexpr int W = 8;
        for (int first = 0; first < end; first += kKeepThreads * W) {
            int from[W];
            float w[W];
#pragma unroll
            for (int u = 0; u < W; ++u) {
                const int i = first + u * kKeepThreads + tid;
                from[u] = i < end ? kept[i] : -1;
            }
#pragma unroll
            for (int u = 0; u < W; ++u) {
                const int i = first + u * kKeepThreads + tid;
                w[u] = from[u] >= i && from[u] < have ? sums[from[u]] : 0.f;
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int u = 0; u < W; ++u) {
                const int i = first + u * kKeepThreads + tid;
                if (i < end) sums[i] = w[u];
            }
        }
        for (int i = end + tid; i < have; i += kKeepThreads) sums[i] = 0.f;     // (every entry of the list has been read)
        return;
    }
    const int l = tid % LANES, mine = tid / LANES, end = a.keep < len ? a.keep : len;
    for (int list = 0; list < end; list += kListed) {
        const int listed = end - list < kListed ? end - list : kListed;
        // (the last batch has left the list behind the barrier between its loads and stores but for its targets, which its threads hold)
#pragma unroll
        for (int u = 0; u < kListed / kKeepThreads; ++u) {
            const int i = list + u * kKeepThreads + tid, source = i < end ? kept[i] : -1;
            const bool moves = source > i && source < len;
            const int from_page = divided(moves ? source : 0, a.pages), to_page = divided(moves ? i : 0, a.pages);
            const bool listed_pages = from_page < npages;
            const int64_t from = c.indices[p0 + (listed_pages ? from_page : 0)], to = c.indices[p0 + (listed_pages ? to_page : 0)];
            const bool good = moves && listed_pages && from >= 0 && from < c.num_pages && to >= 0 && to < c.num_pages;
            sources[u * kKeepThreads + tid] = good ? paged_slot(c, from, side, h, source - from_page * c.page_size) : -1;
            targets[u * kKeepThreads + tid] = good ? paged_slot(c, to, side, h, i - to_page * c.page_size) : -1;
        }
        __syncthreads();
        for (int first = 0; first < listed; first += EACH * TURNS) {
            u32x4 v[TURNS];
            u32 p[TURNS];
            int64_t to[TURNS];
#pragma unroll
            for (int u = 0; u < TURNS; ++u) {
                const int i = first + u * EACH + mine;
                to[u] = i < listed ? targets[i] : -1;
                if (to[u] >= 0) {
                    const int64_t at = sources[i];
                    v[u] = *((const u32x4*)c.data + at * LANES + l);
                    if (l == 0) p[u] = c.param[at];
                }
            }
            // (a batch's loads are over before any of its stores begins)
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int u = 0; u < TURNS; ++u)
                if (to[u] >= 0) {
                    *((u32x4*)c.data + to[u] * LANES + l) = v[u];
                    if (l == 0) c.param[to[u]] = p[u];
                }
        }
    }
}

int keep_positions(bool fp16, const void* kept, int64_t keep, void* kv_data, void* kv_param, const void* kv_indptr, const void* kv_indices, const void* last_page_offset,
                   int64_t num_pages, int num_layers, int layer_idx, int num_heads, int page_size, int head_dim, int64_t batch_size, void* weights, int64_t capacity,
                   void* stream) {
    const int rc = qr_internal_check_paged_cache(kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads, page_size,
                                                 head_dim, batch_size);
    if (rc != QR_OK) return rc;
    if (keep < 0 || keep > 0x3fffffff || capacity < 0) return QR_E_SHAPE;
    if (batch_size == 0) return QR_OK;
    if (batch_size > 0x1fffff || batch_size * num_heads > 0x1fffff) return QR_E_SHAPE;      // (a launch has fewer than 2^32 threads)
    if (keep > 0 && !kept) return QR_E_NULL;
    if (((uintptr_t)kept & 3) || ((uintptr_t)weights & 3)) return QR_E_ALIGN;
    Keep a;
    a.c = qr_internal_paged_kv(kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads, page_size, batch_size);
    a.kept = (const int32_t*)kept;
    a.sums = (float*)weights;
    a.capacity = capacity;
    a.keep = (int)keep;
    a.jobs = weights && capacity > 0 ? 3 : 2;
    a.pages = divisor_of(page_size);
    const dim3 grid((unsigned)(batch_size * num_heads * a.jobs));
    if (fp16) keep_positions_kernel<true><<<grid, dim3(kKeepThreads), 0, (hipStream_t)stream>>>(a);
    else keep_positions_kernel<false><<<grid, dim3(kKeepThreads), 0, (hipStream_t)stream>>>(a);
    return qr_launch_status();
}

}  // namespace

extern "C" int qr_heavy_positions(const void* weights, int64_t capacity, const void* lengths, int64_t batch_size, int num_heads, int64_t keep, int64_t sinks,
                                  int64_t recent, void* kept, void* new_lengths, void* stream) {
    if (batch_size < 0 || num_heads <= 0 || capacity < 0 || capacity > 0x3fffffff || keep < 0 || keep > 0x3fffffff || sinks < 0 || recent < 0 || sinks > keep ||
        recent > keep - sinks)
        return QR_E_SHAPE;
    if (batch_size == 0) return QR_OK;
    if (batch_size > 0x3fffff || batch_size * num_heads > 0x3fffff) return QR_E_SHAPE;      // (a launch has fewer than 2^32 threads)
    if ((!weights && capacity > 0) || !lengths || (!kept && keep > 0) || !new_lengths) return QR_E_NULL;
    if (((uintptr_t)weights & 3) || ((uintptr_t)lengths & 3) || ((uintptr_t)kept & 3) || ((uintptr_t)new_lengths & 3)) return QR_E_ALIGN;
    // (a workgroup per key head reads a sequence's length, and one of them writes the new one)
    const uintptr_t from = (uintptr_t)lengths, to = (uintptr_t)new_lengths, bytes = (uintptr_t)batch_size * 4;
    if (from < to + bytes && to < from + bytes) return QR_E_UNSUPPORTED;
    Heavy a;
    a.sums = (const float*)weights, a.lengths = (const int32_t*)lengths;
    a.kept = (int32_t*)kept, a.left = (int32_t*)new_lengths;
    a.capacity = capacity;
    a.heads = num_heads, a.keep = (int)keep, a.sinks = (int)sinks, a.recent = (int)recent;
    const dim3 grid((unsigned)(batch_size * num_heads)), threads(kHeavyThreads);
    // As few registers as the lists can need (microseconds of 8 lists of 4000 5.2, with eight 6.1, with sixteen 6.7; of 8000 6.5, with sixteen 7.1; of 16000 10.2, with 32 10.1 - 12 where there
    // are more lists); longer ones are read from memory for every digit (60000 52, in 64 registers of which some spill 40, but 1024 lists 174 and 202).
    if (capacity <= 4 * kHeavyThreads) heavy_positions_kernel<4><<<grid, threads, 0, (hipStream_t)stream>>>(a);
    else if (capacity <= 8 * kHeavyThreads) heavy_positions_kernel<8><<<grid, threads, 0, (hipStream_t)stream>>>(a);
    else if (capacity <= 16 * kHeavyThreads) heavy_positions_kernel<16><<<grid, threads, 0, (hipStream_t)stream>>>(a);
    else if (capacity <= 32 * kHeavyThreads) heavy_positions_kernel<32><<<grid, threads, 0, (hipStream_t)stream>>>(a);
    else heavy_positions_kernel<0><<<grid, threads, 0, (hipStream_t)stream>>>(a);
    return qr_launch_status();
}

#define QR_KEEP_ENTRY(NAME, FP16)                                                                                                                        \
    extern "C" int NAME(const void* kept, int64_t keep, void* kv_data, void* kv_param, const void* kv_indptr, const void* kv_indices,                    \
                        const void* last_page_offset, int64_t num_pages, int num_layers, int layer_idx, int num_heads, int page_size, int head_dim,      \
                        int64_t batch_size, void* weights_or_null, int64_t capacity, void* stream) {                                                     \
        return keep_positions(FP16, kept, keep, kv_data, kv_param, kv_indptr, kv_indices, last_page_offset, num_pages, num_layers, layer_idx, num_heads,  \
                              page_size, head_dim, batch_size, weights_or_null, capacity, stream);                                                       \
    }
QR_KEEP_ENTRY(qr_keep_positions_i4, false)
QR_KEEP_ENTRY(qr_keep_positions_f16, true)
