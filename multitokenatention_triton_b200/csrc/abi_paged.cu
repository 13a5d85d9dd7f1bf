// C entry points of the paged cache and of the attention that reads it: argument checks, then the launchers.
#include "paged.cuh"

namespace mta {
namespace {

// The checks that all calls over a cache share; fills `c`.  K is the call's name in messages.
int describe(PagedCache* c, const char* K, const void* q_hist, const void* k, const void* v, const int* table, const int* lengths, const int* slot_ids, int slots,
             int table_width, int pages, int page, int ring, int H, int kv_heads, int D, int max_length, int B, int dtype) {
    MTA_REQUIRE(dtype_ok(dtype), "%s: unknown dtype code %d", K, dtype);
    MTA_REQUIRE(B >= 0 && slots >= 1 && table_width >= 1 && pages >= 1 && ring >= 1, "%s: bad cache: %d rows, %d slots of %d pages, %d pages, %d queries", K, B,
                slots, table_width, pages, ring);
    MTA_REQUIRE(slot_ids || B <= slots, "%s: %d batch rows, but the cache has %d slots", K, B, slots);
    MTA_REQUIRE(H >= 1 && kv_heads >= 1 && H % kv_heads == 0, "%s: %d heads are no multiple of %d key-value heads", K, H, kv_heads);
    MTA_REQUIRE(page >= 16 && page <= 65536 && (page & (page - 1)) == 0, "%s: a page of %d tokens; a power of two from 16 to 65536 is wanted", K, page);
    const int most = dtype == MTA_F32 ? 128 : 256;
    MTA_REQUIRE(D >= 8 && D % 8 == 0 && D <= most, "%s: head dimension %d; a multiple of 8 up to %d is wanted", K, D, most);
    MTA_REQUIRE(max_length >= 0 && max_length <= (long)table_width * page, "%s: a longest sequence of %d tokens, but a table row holds %ld", K, max_length,
                (long)table_width * page);
    MTA_REQUIRE((long)table_width * page <= 1L << 30, "%s: table rows of %d pages of %d tokens; sequences of up to 2^30 tokens are supported", K, table_width, page);
    MTA_REQUIRE(q_hist && k && v && table && lengths, "%s: null pointer", K);
    MTA_REQUIRE(aligned16(q_hist) && aligned16(k) && aligned16(v), "%s: queries, keys and values must begin on 16-byte boundaries", K);
    c->q_hist = q_hist; c->k = k; c->v = v; c->table = table; c->lengths = lengths; c->slot_ids = slot_ids;
    c->slots = slots; c->table_width = table_width; c->pages = pages; c->ring = ring; c->H = H; c->kv_heads = kv_heads; c->D = D;
    c->page_shift = 0;
    while (1 << c->page_shift < page) ++c->page_shift;
    c->max_length = max_length;
    c->err = nullptr;
    return MTA_OK;
}

int check_taps(const char* K, int cq, int ck, int rows) {
    MTA_REQUIRE(cq >= 1 && ck >= 1 && ck <= DECODE_MAX_TAPS, "%s: kernel %dx%d; 1 to %d key taps are supported", K, cq, ck, DECODE_MAX_TAPS);
    MTA_REQUIRE(cq <= DECODE_MAX_ROWS && rows <= DECODE_MAX_ROWS, "%s: a token looks at %d queries; at most %d are supported", K, rows, DECODE_MAX_ROWS);
    return MTA_OK;
}

int check_ring(const char* K, int rows, int ring) {
    MTA_REQUIRE(rows <= ring, "%s: a token looks at %d queries, but the cache keeps %d", K, rows, ring);
    return MTA_OK;
}

int check_batch(const char* K, int B, int max_length) {
    MTA_REQUIRE(B <= DECODE_MAX_BATCH, "%s: %d batch rows; at most %d are supported in one call", K, B, DECODE_MAX_BATCH);
    MTA_REQUIRE((long)B * max_length <= 1L << 34, "%s: %d rows of up to %d tokens; at most 2^34 tokens together are supported", K, B, max_length);
    return MTA_OK;
}

// What the shapes alone decide, of calls that the workspace sizes are asked for.
int check_sizes(const char* K, int B, int H, int kv_heads, int D, int max_length) {
    MTA_REQUIRE(B >= 0 && H >= 1 && kv_heads >= 1 && H % kv_heads == 0 && D >= 8 && max_length >= 0, "%s: bad sizes: %d rows, %d heads on %d of %d elements, %d tokens", K,
                B, H, kv_heads, D, max_length);
    return check_batch(K, B, max_length);
}
int conv_attn_size(const char* K, int B, int H, int kv_heads, int D, int cq, int ck, int max_length, size_t* bytes) {
    if (int rc = check_sizes(K, B, H, kv_heads, D, max_length)) return rc;
    if (int rc = check_taps(K, cq, ck, cq)) return rc;
    *bytes = conv_attn_decode_workspace(B, H, kv_heads, D, cq, max_length);
    return MTA_OK;
}
int mta_size(const char* K, int B, int H, int kv_heads, int D, int cq, int ck, int cq2, int ck2, int max_length, size_t* bytes) {
    if (int rc = check_sizes(K, B, H, kv_heads, D, max_length)) return rc;
    MTA_REQUIRE(H <= 128, "%s: %d heads; at most 128 are supported", K, H);
    MTA_REQUIRE(cq2 >= 1 && cq2 <= DECODE_MAX_ROWS && cq <= DECODE_MAX_ROWS, "%s: %d and %d query taps", K, cq, cq2);
    if (int rc = check_taps(K, cq, ck, cq + cq2 - 1)) return rc;
    if (int rc = check_taps(K, cq2, ck2, cq + cq2 - 1)) return rc;
    return mta_decode_workspace(B, H, kv_heads, D, cq, ck, cq2, ck2, max_length, bytes);
}
}  // namespace
}  // namespace mta

using namespace mta;

extern "C" {

int mta_cache_append(const void* k, const void* v, const void* q, const long long* strides, const int* counts, void* k_pages, void* v_pages, void* q_hist,
                     const int* table, const int* lengths, const int* slot_ids, int B, int T, int slots, int table_width, int pages, int page, int ring, int H,
                     int kv_heads, int D, int dtype, void* stream) {
    set_error("%s", "");
    PagedCache c;
    MTA_REQUIRE(T >= 0, "cache_append: %d tokens", T);
    MTA_REQUIRE(table_width >= 1 && page >= 1 && (long)table_width * page <= 0x7fffffffL, "cache_append: rows of %d pages of %d tokens", table_width, page);
    if (int rc = describe(&c, "cache_append", q_hist, k_pages, v_pages, table, lengths, slot_ids, slots, table_width, pages, page, ring, H, kv_heads, D,
                          table_width * page, B, dtype)) return rc;
    if ((long)B * T == 0) return MTA_OK;
    MTA_REQUIRE(k && v && q && strides, "cache_append: null pointer");
    MTA_REQUIRE(aligned16(k) && aligned16(v) && aligned16(q), "cache_append: k, v and q must begin on 16-byte boundaries");
    long s[9];
    for (int i = 0; i < 9; ++i) {
        s[i] = (long)strides[i];
        MTA_REQUIRE(s[i] * (long)dtype_size(dtype) % 16 == 0, "cache_append: stride %ld is no multiple of 16 bytes", s[i]);
    }
    if (int rc = check_device()) return rc;
    return cache_append_launch(c, k, v, q, s, counts, B, T, dtype, static_cast<cudaStream_t>(stream));
}

int mta_cache_status(void* stream) {
    set_error("%s", "");
    int* flag = nullptr;
    if (int rc = wait_flag_ptr(&flag)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int raised = 0;
    MTA_CUDA_OK(cudaMemcpyAsync(&raised, flag + 1, sizeof(int), cudaMemcpyDeviceToHost, st));
    MTA_CUDA_OK(cudaStreamSynchronize(st));
    if (!raised) return MTA_OK;
    MTA_CUDA_OK(cudaMemsetAsync(flag + 1, 0, sizeof(int), st));
    MTA_CUDA_OK(cudaStreamSynchronize(st));
    set_error("a cache call since the last check met a page, slot, length or count out of range: what it named was neither read nor written");
    return MTA_ERR_INVALID;
}

int mta_cache_copy(void* k_pages, void* v_pages, const int* src, const int* dst, int n, long long page_bytes, int pages, void* q_hist, const int* slot_src,
                   const int* slot_dst, int n_slots, long long slot_bytes, int slots, int layers, void* stream) {
    set_error("%s", "");
    MTA_REQUIRE(n >= 0 && n_slots >= 0 && layers >= 1 && layers <= 16384, "cache_copy: bad sizes: %d pages, %d slots, %d layers", n, n_slots, layers);
    if (n == 0 && n_slots == 0) return MTA_OK;
    MTA_REQUIRE(n == 0 || (k_pages && v_pages && src && dst), "cache_copy: null pointer");
    MTA_REQUIRE(n_slots == 0 || (q_hist && slot_src && slot_dst), "cache_copy: null pointer");
    MTA_REQUIRE(n == 0 || (page_bytes > 0 && page_bytes % 16 == 0 && page_bytes <= 1LL << 30 && pages >= 1 && aligned16(k_pages) && aligned16(v_pages)),
                "cache_copy: %d pages of %lld bytes; 16-byte aligned pages of a multiple of 16 bytes up to 1 GiB are wanted", pages, page_bytes);
    MTA_REQUIRE(n_slots == 0 || (slot_bytes > 0 && slot_bytes % 16 == 0 && slot_bytes <= 1LL << 30 && slots >= 1 && aligned16(q_hist)),
                "cache_copy: %d slots of %lld bytes; 16-byte aligned slots of a multiple of 16 bytes up to 1 GiB are wanted", slots, slot_bytes);
    if (int rc = check_device()) return rc;
    return cache_copy_launch(k_pages, v_pages, src, dst, n, n ? page_bytes : 0, pages, q_hist, slot_src, slot_dst, n_slots, n_slots ? slot_bytes : 0, slots, layers,
                             static_cast<cudaStream_t>(stream));
}

size_t mta_conv_attn_decode_workspace_bytes(int B, int H, int kv_heads, int D, int cq, int ck, int max_length) {
    set_error("%s", "");
    size_t bytes = 0;
    return conv_attn_size("conv_attn_decode", B, H, kv_heads, D, cq, ck, max_length, &bytes) ? 0 : bytes;
}

int mta_conv_attn_decode_fwd(const void* q_hist, const void* k_pages, const void* v_pages, const int* table, const int* lengths, const int* slot_ids, const void* w,
                             void* o, void* workspace, size_t workspace_bytes, int B, int slots, int table_width, int pages, int page, int ring, int H,
                             int kv_heads, int D, int cq, int ck, int max_length, float scale, int dtype, int w_dtype, void* stream) {
    set_error("%s", "");
    PagedCache c;
    const char* K = "conv_attn_decode";
    if (int rc = describe(&c, K, q_hist, k_pages, v_pages, table, lengths, slot_ids, slots, table_width, pages, page, ring, H, kv_heads, D, max_length, B, dtype))
        return rc;
    MTA_REQUIRE(dtype_ok(w_dtype), "%s: unknown dtype code %d of the weight", K, w_dtype);
    size_t need = 0;
    if (int rc = conv_attn_size(K, B, H, kv_heads, D, cq, ck, max_length, &need)) return rc;
    if (int rc = check_ring(K, cq, ring)) return rc;
    if (B == 0) return MTA_OK;
    MTA_REQUIRE(w && o && aligned16(o), "%s: null or unaligned pointer", K);
    MTA_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, "%s: workspace of %zu bytes (16-byte aligned) is smaller than the %zu needed", K,
                workspace_bytes, need);
    if (int rc = check_device()) return rc;
    return conv_attn_decode_launch(c, w, w_dtype, o, workspace, B, cq, ck, scale, dtype, static_cast<cudaStream_t>(stream));
}

size_t mta_decode_workspace_bytes(int B, int H, int kv_heads, int D, int cq, int ck, int cq2, int ck2, int max_length) {
    set_error("%s", "");
    size_t bytes = 0;
    return mta_size("mta_decode", B, H, kv_heads, D, cq, ck, cq2, ck2, max_length, &bytes) ? 0 : bytes;
}

int mta_decode_fwd(const void* q_hist, const void* k_pages, const void* v_pages, const int* table, const int* lengths, const int* slot_ids, const void* w1,
                   const void* W1, const void* w2, const void* W2, void* o, void* workspace, size_t workspace_bytes, int B, int slots, int table_width, int pages,
                   int page, int ring, int H, int kv_heads, int D, int cq, int ck, int cq2, int ck2, int max_length, int dtype, int w_dtype, void* stream) {
    set_error("%s", "");
    PagedCache c;
    const char* K = "mta_decode";
    if (int rc = describe(&c, K, q_hist, k_pages, v_pages, table, lengths, slot_ids, slots, table_width, pages, page, ring, H, kv_heads, D, max_length, B, dtype))
        return rc;
    MTA_REQUIRE(dtype_ok(w_dtype), "%s: unknown dtype code %d of the weights", K, w_dtype);
    size_t need = 0;
    if (int rc = mta_size(K, B, H, kv_heads, D, cq, ck, cq2, ck2, max_length, &need)) return rc;
    if (int rc = check_ring(K, cq + cq2 - 1, ring)) return rc;
    if (B == 0) return MTA_OK;
    MTA_REQUIRE(w1 && W1 && w2 && W2 && o, "%s: null pointer", K);
    MTA_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, "%s: workspace of %zu bytes (16-byte aligned) is smaller than the %zu needed", K,
                workspace_bytes, need);
    if (int rc = check_device()) return rc;
    return mta_decode_launch(c, w1, W1, w2, W2, w_dtype, o, workspace, B, cq, ck, cq2, ck2, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
