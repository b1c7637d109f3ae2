// Page tables of a batch whose sequences differ in length, and places of their new tokens, from lengths that lie on the GPU.
#include "qr_common.h"

namespace {

struct Tables {
    const int32_t* lengths;
    const int32_t* fresh;             // nullptr: no new tokens are asked about
    const int32_t* block_table;       // nullptr: page i of sequence b is page number i * batch + b
    int32_t* indptr;
    int32_t* indices;
    int32_t* last;
    int32_t* starts;
    int64_t* positions;
    int64_t* slots;
    int64_t table_stride, tokens, capacity;
    int batch, page_size, max_pages, each, groups;         // sequences of a workgroup, workgroups
};

__device__ __forceinline__ int held(const Tables& t, int b) {           // tokens of sequence b: no more than its pages hold
    const int64_t most = (int64_t)t.max_pages * t.page_size;
    const int n = t.lengths[b];
    return n < 0 ? 0 : n > most ? (int)most : n;
}
__device__ __forceinline__ int pages_of(const Tables& t, int n) { return (int)(((int64_t)n + t.page_size - 1) / t.page_size); }

// One workgroup per sequence, or per t.each sequences that follow one another where there are more than kGroups.  Each adds up the page counts and new tokens of the
// sequences before its own by itself (a batch of 512 is two loads per thread), so there is one launch and no workgroup waits for another; with a workgroup per
// sequence whatever their number the loads would grow by its square.
constexpr int kGroups = 2048;
__global__ __launch_bounds__(256) void build_page_tables_kernel(Tables t) {
    __shared__ int sums[4][2];
    __shared__ int64_t token_sums[4][2];
    const int first = blockIdx.x * t.each, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int before = 0, all = 0;                               // (the host has seen that all pages' entries are counted in 32 bits; new tokens may be any number)
    int64_t tokens_before = 0, tokens_all = 0;
    for (int i = threadIdx.x; i < t.batch; i += 256) {
        const int p = pages_of(t, held(t, i));
        all += p;
        before += i < first ? p : 0;
        if (t.fresh) {
            const int n = t.fresh[i] < 0 ? 0 : t.fresh[i];
            tokens_all += n;
            tokens_before += i < first ? n : 0;
        }
    }
#pragma unroll
    for (int mask = 1; mask < 64; mask *= 2) {
        before += __shfl_xor(before, mask, 64);
        all += __shfl_xor(all, mask, 64);
        tokens_before += __shfl_xor(tokens_before, mask, 64);
        tokens_all += __shfl_xor(tokens_all, mask, 64);
    }
    if (lane == 0) sums[wave][0] = before, sums[wave][1] = all, token_sums[wave][0] = tokens_before, token_sums[wave][1] = tokens_all;
    __syncthreads();
    before = sums[0][0] + sums[1][0] + sums[2][0] + sums[3][0];
    all = sums[0][1] + sums[1][1] + sums[2][1] + sums[3][1];
    tokens_before = token_sums[0][0] + token_sums[1][0] + token_sums[2][0] + token_sums[3][0];
    tokens_all = token_sums[0][1] + token_sums[1][1] + token_sums[2][1] + token_sums[3][1];

    auto bound = [](int64_t tokens) { return (int)(tokens > 0x7fffffff ? 0x7fffffff : tokens); };        // (behind all tokens that there are)
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        t.indptr[t.batch] = all;
        if (t.starts) t.starts[t.batch] = bound(tokens_all);
    }
    const int64_t thread = (int64_t)blockIdx.x * 256 + threadIdx.x, threads = (int64_t)t.groups * 256;
    for (int64_t i = all + thread; i < t.capacity; i += threads) t.indices[i] = -1;
    if (t.fresh)
        for (int64_t i = tokens_all + thread; i < t.tokens; i += threads) t.positions[i] = t.slots[i] = -1;

    for (int b = first; b < t.batch && b < first + t.each; ++b) {
        const int n = held(t, b), pages = pages_of(t, n);
        auto page_at = [&](int i) { return t.block_table ? t.block_table[b * t.table_stride + i] : i * t.batch + b; };
        if (threadIdx.x == 0) {
            t.indptr[b] = before;
            t.last[b] = n > 0 ? n - (pages - 1) * t.page_size : 0;
            if (t.starts) t.starts[b] = bound(tokens_before);
        }
        for (int i = threadIdx.x; i < pages; i += 256) t.indices[(int64_t)before + i] = page_at(i);
        before += pages;
        if (!t.fresh) continue;
        const int fresh = t.fresh[b] < 0 ? 0 : t.fresh[b];
        for (int i = threadIdx.x; i < fresh && tokens_before + i < t.tokens; i += 256) {
            const int pos = n - fresh + i;
            t.positions[tokens_before + i] = pos;
            int64_t slot = -1;
            if (pos >= 0) {
                const int it = pos / t.page_size, page = page_at(it);
                if (page >= 0) slot = (int64_t)page * t.page_size + (pos - it * t.page_size);
            }
            t.slots[tokens_before + i] = slot;
        }
        tokens_before += fresh;
    }
}

}  // namespace

extern "C" int qr_build_page_tables(const void* lengths, const void* new_lengths_or_null, int64_t batch_size, int page_size, int64_t max_pages,
                                    const void* block_table_or_null, int64_t table_stride, int64_t tokens, void* kv_indptr, void* kv_indices,
                                    void* last_page_offset, void* seqlen_indptr, void* positions, void* slots, void* stream) {
    if (batch_size < 0 || page_size <= 0 || max_pages <= 0 || tokens < 0 || tokens > 0x3fffffff) return QR_E_SHAPE;        // (counted in 32 bits)
    if (batch_size == 0) return QR_OK;
    if (batch_size > 0x3fffffff || max_pages > 0x3fffffff || max_pages * batch_size > 0x3fffffff || max_pages * page_size > 0x7fffffff) return QR_E_SHAPE;
    if (block_table_or_null && table_stride < max_pages) return QR_E_SHAPE;
    if (!lengths || !kv_indptr || !kv_indices || !last_page_offset) return QR_E_NULL;
    if (new_lengths_or_null ? (!seqlen_indptr || (tokens > 0 && (!positions || !slots))) : tokens > 0) return new_lengths_or_null ? QR_E_NULL : QR_E_SHAPE;
    Tables t;
    t.lengths = (const int32_t*)lengths;
    t.fresh = (const int32_t*)new_lengths_or_null;
    t.block_table = (const int32_t*)block_table_or_null;
    t.indptr = (int32_t*)kv_indptr;
    t.indices = (int32_t*)kv_indices;
    t.last = (int32_t*)last_page_offset;
    t.starts = (int32_t*)(new_lengths_or_null ? seqlen_indptr : nullptr);
    t.positions = (int64_t*)positions;
    t.slots = (int64_t*)slots;
    t.table_stride = table_stride, t.tokens = tokens, t.capacity = batch_size * max_pages;
    t.batch = (int)batch_size, t.page_size = page_size, t.max_pages = (int)max_pages;
    t.each = (int)((batch_size + kGroups - 1) / kGroups), t.groups = (int)((batch_size + t.each - 1) / t.each);
    build_page_tables_kernel<<<dim3((unsigned)t.groups), dim3(256), 0, (hipStream_t)stream>>>(t);
    return qr_launch_status();
}
