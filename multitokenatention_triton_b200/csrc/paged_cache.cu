// Writes into a paged cache: new tokens' keys, values and queries, and copies of whole pages.  Both only move bytes, and HBM bounds
// them: prompts of 8 x up to 4096 tokens, 16 heads of 128 in bf16 64 us = 5.9 TB/s read and written, 1500 pages of 64 tokens 241 us = 6.5 TB/s;
// one token of 64 sequences 2.2 us, eight pages 2.4 us, their launches.
#include "paged.cuh"

namespace mta {
namespace {

struct AppendArgs {
    const uint4 *k, *v, *q;               // (B, heads, T, D) with strides in 16-byte vectors
    long ks[3], vs[3], qs[3];
    uint4 *k_pages, *v_pages, *q_hist;
    const int* counts;                    // tokens of each batch row, null: T
    int T, vecs;                          // 16-byte vectors in a row
};

// One thread per 16-byte vector of K and of V, or of the queries: source and destination are contiguous along a head's tokens, so
// neighbouring threads read and write neighbouring addresses.  Indices are 32-bit: the host refuses more vectors.
__global__ void __launch_bounds__(256) cache_append_kernel(PagedCache c, AppendArgs a, unsigned kv_items, unsigned q_items, int q_rows) {
    pdl_wait();
    const unsigned step = gridDim.x * blockDim.x;
    const int page_mask = (1 << c.page_shift) - 1;
    for (unsigned i = blockIdx.x * blockDim.x + threadIdx.x; i < kv_items + q_items; i += step) {
        const bool kv = i < kv_items;
        unsigned x = kv ? i : i - kv_items;
        const int heads = kv ? c.kv_heads : c.H, rows = kv ? a.T : q_rows;
        const int vec = x % a.vecs; x /= a.vecs;
        const int row = x % rows; x /= rows;
        const int h = x % heads, b = x / heads;
        const int slot = c.slot(b);
        if ((unsigned)slot >= (unsigned)c.slots) { c.bad(); continue; }
        const int n = a.counts ? __ldg(a.counts + b) : a.T, len = __ldg(c.lengths + slot);
        if (n < 0 || n > a.T || len < n || len > c.max_length) { c.bad(); continue; }
        // of the queries only the last `ring` are kept
        const int token = kv ? row : n - q_rows + row;
        if (token < 0 || token >= n) continue;
        const int pos = len - n + token;
        if (kv) {
            const int p = __ldg(c.table + (long)slot * c.table_width + (pos >> c.page_shift));
            if ((unsigned)p >= (unsigned)c.pages) { c.bad(); continue; }
            const long to = ((((long)p * c.kv_heads + h) << c.page_shift) + (pos & page_mask)) * a.vecs + vec;
            a.k_pages[to] = __ldg(a.k + b * a.ks[0] + h * a.ks[1] + token * a.ks[2] + vec);
            a.v_pages[to] = __ldg(a.v + b * a.vs[0] + h * a.vs[1] + token * a.vs[2] + vec);
        } else {
            const long to = (((long)slot * c.ring + pos % c.ring) * c.H + h) * a.vecs + vec;
            a.q_hist[to] = __ldg(a.q + b * a.qs[0] + h * a.qs[1] + token * a.qs[2] + vec);
        }
    }
}

struct CopyPool {
    uint4* base;
    const int *src, *dst;
    long vecs;                            // 16-byte vectors of one block (page or ring)
    int n, blocks;                        // pairs; blocks of one layer
};

constexpr int COPY_VECS = 8;              // per thread, all in flight at once
constexpr int COPY_THREADS = 256;

// Grid: (pairs, parts of a block, pool and layer).  Pairs that name a block outside the pool are skipped.
__global__ void __launch_bounds__(COPY_THREADS) cache_copy_kernel(CopyPool k, CopyPool v, CopyPool q, int layers, int* err) {
    pdl_wait();
    const int pool = blockIdx.z / layers, layer = blockIdx.z % layers;
    const CopyPool p = pool == 0 ? k : pool == 1 ? v : q;
    const long first = (long)blockIdx.y * COPY_VECS * COPY_THREADS + threadIdx.x;
    if ((int)blockIdx.x >= p.n || (long)blockIdx.y * COPY_VECS * COPY_THREADS >= p.vecs) return;
    const int s = __ldg(p.src + blockIdx.x), d = __ldg(p.dst + blockIdx.x);
    if ((unsigned)s >= (unsigned)p.blocks || (unsigned)d >= (unsigned)p.blocks) {
        if (threadIdx.x == 0) atomicExch(err + 1, 1);
        return;
    }
    const uint4* from = p.base + ((long)layer * p.blocks + s) * p.vecs;
    uint4* to = p.base + ((long)layer * p.blocks + d) * p.vecs;
    uint4 r[COPY_VECS];
#pragma unroll
    for (int i = 0; i < COPY_VECS; ++i)
        if (first + i * COPY_THREADS < p.vecs) r[i] = from[first + i * COPY_THREADS];
#pragma unroll
    for (int i = 0; i < COPY_VECS; ++i)
        if (first + i * COPY_THREADS < p.vecs) to[first + i * COPY_THREADS] = r[i];
}

}  // namespace

int cache_append_launch(const PagedCache& cache, const void* k, const void* v, const void* q, const long* strides, const int* counts, int B, int T,
                        int dtype, cudaStream_t st) {
    PagedCache c = cache;
    if (int rc = wait_flag_ptr(&c.err)) return rc;
    const int epv = 16 / (int)dtype_size(dtype);
    AppendArgs a;
    a.k = static_cast<const uint4*>(k); a.v = static_cast<const uint4*>(v); a.q = static_cast<const uint4*>(q);
    for (int i = 0; i < 3; ++i) { a.ks[i] = strides[i] / epv; a.vs[i] = strides[3 + i] / epv; a.qs[i] = strides[6 + i] / epv; }
    a.k_pages = static_cast<uint4*>(const_cast<void*>(c.k)); a.v_pages = static_cast<uint4*>(const_cast<void*>(c.v));
    a.q_hist = static_cast<uint4*>(const_cast<void*>(c.q_hist));
    a.counts = counts; a.T = T; a.vecs = c.D / epv;
    const int q_rows = T < c.ring ? T : c.ring;
    const long kv = (long)B * c.kv_heads * T * a.vecs, qi = (long)B * c.H * q_rows * a.vecs;
    MTA_REQUIRE(kv + qi < (1L << 31), "cache_append: %ld vectors of 16 bytes in one call exceed %ld: append in parts", kv + qi, (1L << 31) - 1);
    int sms = 0;
    if (int rc = sm_count(&sms)) return rc;
    long blocks = (kv + qi + 255) / 256;
    if (blocks > (long)sms * 16) blocks = (long)sms * 16;
    return launch_kernel<cache_append_kernel>("cache_append_kernel", dim3((unsigned)blocks), 256, 0, st, c, a, (unsigned)kv, (unsigned)qi, q_rows);
}

int cache_copy_launch(void* k_pages, void* v_pages, const int* src, const int* dst, int n, long page_bytes, int pages, void* q_hist, const int* slot_src,
                      const int* slot_dst, int n_slots, long slot_bytes, int slots, int layers, cudaStream_t st) {
    int* err = nullptr;
    if (int rc = wait_flag_ptr(&err)) return rc;
    const CopyPool k{static_cast<uint4*>(k_pages), src, dst, page_bytes / 16, n, pages}, v{static_cast<uint4*>(v_pages), src, dst, page_bytes / 16, n, pages};
    const CopyPool q{static_cast<uint4*>(q_hist), slot_src, slot_dst, slot_bytes / 16, n_slots, slots};
    const long per = COPY_VECS * COPY_THREADS;
    const long vecs = n && (!n_slots || k.vecs > q.vecs) ? k.vecs : q.vecs;
    const dim3 grid((unsigned)(n > n_slots ? n : n_slots), (unsigned)((vecs + per - 1) / per), (unsigned)((n_slots ? 3 : 2) * layers));
    return launch_kernel<cache_copy_kernel>("cache_copy_kernel", grid, COPY_THREADS, 0, st, k, v, q, layers, err);
}

}  // namespace mta
