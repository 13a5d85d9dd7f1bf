// What the kernels over a paged cache share: the cache's description, the bounds checks of what it says, and the tiles of 16 keys
// and values that a warp holds in registers.
#pragma once

#include "kernels.cuh"
#include "tc05.cuh"

namespace mta {

// A paged cache of one layer.  k, v: (pages, kv_heads, page, D); q_hist: (slots, ring, H, D), the query of position p at p % ring;
// table: (slots, table_width) page numbers; lengths: (slots) tokens, the newest among them.  Batch row b is slot slot_ids[b] (b when
// null).  `page` is a power of two from 16 on, so that 16 keys from a multiple of 16 on lie in one page.
struct PagedCache {
    const void* q_hist;
    const void* k;
    const void* v;
    const int* table;
    const int* lengths;
    const int* slot_ids;
    int slots, table_width, pages, page_shift, ring, H, kv_heads, D;
    int max_length;      // no sequence of the call is longer
    int* err;            // the device's flags: [1] is raised by what a table, length or slot says wrongly

    // Raises the flag of a bad table, length or slot: that part of the cache is not touched, mta_cache_status() reports it.
    __device__ void bad() const { atomicExch(err + 1, 1); }
    __device__ int slot(int b) const { return slot_ids ? __ldg(slot_ids + b) : b; }
    // Tokens of batch row b; 0 where slot or length are out of range.
    __device__ int length(int b) const {
        const int s = slot(b);
        if ((unsigned)s >= (unsigned)slots) { bad(); return 0; }
        const int n = __ldg(lengths + s);
        if (n < 0 || n > max_length) { bad(); return 0; }
        return n;
    }
    // Element offset of (kv head, token) in the pools for a slot in range; -1 where the table names no page.
    __device__ long at(int s, int kv_head, int token) const {
        const int p = __ldg(table + (long)s * table_width + (token >> page_shift));
        if ((unsigned)p >= (unsigned)pages) { bad(); return -1; }
        return ((((long)p * kv_heads + kv_head) << page_shift) + (token & ((1 << page_shift) - 1))) * D;
    }
};

constexpr int KEYS = 16;                 // keys of a tile: the columns of two mma.sync, the k index of one
constexpr float LOG2E = 1.4426950408889634f;

template <typename T> __device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 or 32 bytes that are read once: past L1, which keeps the queries.
__device__ __forceinline__ uint4 load_once(const void* p) {
    uint4 r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}
__device__ __forceinline__ void load_once(const void* p, uint4& a, uint4& b) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "l"(p));
}
__device__ __forceinline__ bool aligned32(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 31) == 0; }

// 16 keys of one head in a warp's registers, DMAX >= D elements each.  Lane (g, t) = (lane / 4, lane % 4) holds of rows g and g + 8
// 32 bytes at 128 p + 32 t, as chunks 2p and 2p + 1: one load each, four lanes on a whole line.  An mma sums over its k index in
// any order, so the elements of a lane's 16 bytes may stand for any k as long as the queries are read the same way.  The keys are the
// B operand, two neighbouring registers of a load each; as the A operand, whose four registers come from two loads, every mma cost
// seven moves beside it.  (32-byte loads instead of 16-byte ones: 505 -> 487 us for the MTA step of 16 sequences of 8192 tokens.)
template <typename T, int DMAX> struct KeyTile {
    static constexpr int CH = DMAX * (int)sizeof(T) / 64;
    static constexpr int EPL = 16 / (int)sizeof(T);      // elements in 16 bytes
    static constexpr bool HALF = sizeof(T) == 2;
    // Scores of ROWS query rows (a multiple of 8) in a lane's registers: value i of part p belongs to query row row_of(p, i) and key
    // key_of(p, i) of the tile.
    template <int ROWS> static constexpr int PARTS = HALF ? (ROWS + 15) / 16 * 2 : ROWS / 8;
    static __device__ __forceinline__ int row_of(int p, int i, int lane) { return HALF ? p / 2 * 16 + (lane >> 2) + (i >> 1) * 8 : p * 8 + 2 * (lane & 3) + (i & 1); }
    static __device__ __forceinline__ int key_of(int p, int i, int lane) { return HALF ? p % 2 * 8 + 2 * (lane & 3) + (i & 1) : (lane >> 2) + 8 * (i >> 1); }
    static __device__ __forceinline__ int element(int c, int t) { return (c / 2 * 8 + t * 2 + c % 2) * EPL; }
    uint4 r[2][CH];

    // Rows base, base + 1, ... of which `live` exist; the others are zero and not read.  base < 0: none exists.  The usual whole tile
    // takes a path of plain loads: setting the registers to zero first costs as much as everything else here.
    __device__ __forceinline__ void load(const T* pool, long base, int live, int D, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const T* first = pool + base;
        if (base >= 0 && live >= KEYS && D == DMAX && aligned32(first)) {
            const T* row = first + (g * DMAX + t * 2 * EPL);
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int c = 0; c < CH; c += 2) load_once(row + x * 8 * DMAX + c * 4 * EPL, r[x][c], r[x][c + 1]);
            return;
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const bool on = base >= 0 && g + 8 * x < live;
            const T* row = pool + (on ? base + (long)(g + 8 * x) * D : 0);
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int e = element(c, t);
                r[x][c] = make_uint4(0, 0, 0, 0);
                if (on && e < D) r[x][c] = load_once(row + e);
            }
        }
    }

    // 16 bits: q(m, x) gives the A registers of query rows 16m + g and 16m + g + 8 for the two halves x = 2c, 2c + 1 of chunk c:
    // {row g, row g + 8} of the half's first four bytes, then of its second.  float32: q(row, c) gives 16 bytes (chunk c, position t) of a row.
    template <int ROWS, typename Q> __device__ __forceinline__ void score(float (&acc)[PARTS<ROWS>][4], int lane, Q q) const {
        if constexpr (HALF) {
#pragma unroll
            for (int m = 0; m < PARTS<ROWS> / 2; ++m) {
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[2 * m][i] = acc[2 * m + 1][i] = 0.0f;
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const uint4 a0 = q(m, 2 * c), a1 = q(m, 2 * c + 1);
                    mma_16816<T>(acc[2 * m], a0.x, a0.y, a0.z, a0.w, r[0][c].x, r[0][c].y);
                    mma_16816<T>(acc[2 * m + 1], a0.x, a0.y, a0.z, a0.w, r[1][c].x, r[1][c].y);
                    mma_16816<T>(acc[2 * m], a1.x, a1.y, a1.z, a1.w, r[0][c].z, r[0][c].w);
                    mma_16816<T>(acc[2 * m + 1], a1.x, a1.y, a1.z, a1.w, r[1][c].z, r[1][c].w);
                }
            }
        } else {
            // float32 on FMAs: each lane sums its quarter of the elements for four rows at a time, then the four lanes of a key add up
            // and share out the rows, so that every lane has the two that the mma layout gives it
            const int t = lane & 3;
#pragma unroll
            for (int n = 0; n < PARTS<ROWS>; ++n) {
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float2 p[2][4];                          // sums of even and odd elements
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[0][j] = p[1][j] = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint4 b = q(8 * n + 4 * half + j, c);
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                p[x][j] = __ffma2_rn(make_float2(__uint_as_float(r[x][c].x), __uint_as_float(r[x][c].y)),
                                                     make_float2(__uint_as_float(b.x), __uint_as_float(b.y)), p[x][j]);
                                p[x][j] = __ffma2_rn(make_float2(__uint_as_float(r[x][c].z), __uint_as_float(r[x][c].w)),
                                                     make_float2(__uint_as_float(b.z), __uint_as_float(b.w)), p[x][j]);
                            }
                        }
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float f[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            f[j] = p[x][j].x + p[x][j].y;
                            f[j] += __shfl_xor_sync(0xffffffffu, f[j], 2);
                        }
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float give = t & 1 ? f[j] : f[j + 2], keep = t & 1 ? f[j + 2] : f[j];
                            const float sum = keep + __shfl_xor_sync(0xffffffffu, give, 1);
                            if (t >> 1 == half) acc[n][2 * x + j] = sum;
                        }
                    }
                }
            }
        }
    }
};

// 16 bytes as floats.
__device__ __forceinline__ void unpack16(uint4 u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}

// 16 float32 values of one head in a warp's registers: ROWLANES lanes side by side hold a row, the warp SUBS rows at a time; the
// product with the weights runs on FMAs.
template <int DMAX> struct ValueTileF32 {
    static constexpr int ROWLANES = DMAX / 4, SUBS = 32 / ROWLANES, STEPS = KEYS / SUBS;
    uint4 r[STEPS];

    __device__ __forceinline__ void load(const float* pool, long base, int live, int D, int lane) {
        const int sub = lane / ROWLANES, e = (lane % ROWLANES) * 4;
        if (base >= 0 && live >= KEYS && D == DMAX) {
            const float* row = pool + base + (sub * DMAX + e);
#pragma unroll
            for (int i = 0; i < STEPS; ++i) r[i] = load_once((row + i * SUBS * DMAX));
            return;
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            r[i] = make_uint4(0, 0, 0, 0);
            if (base >= 0 && i * SUBS + sub < live && e < D) r[i] = load_once((pool + base + (long)(i * SUBS + sub) * D + e));
        }
    }
};

// 16 values of one head in 16 bits as the A operand of mma.sync, transposed: rows are elements, columns keys.  Lane (g, t) loads
// 32 bytes at 256 p + 32 g, as chunks 2p and 2p + 1 (DMAX 64: 16 bytes at 16 g), of keys 2t, 2t + 1, 2t + 8 and 2t + 9, and pairs neighbouring keys'
// halves with one byte permute each; mma (c, j) has element e + j as its row g and e + j + 4 as its row g + 8, e = element(c, g).
//
// The B operand's eight columns hold the weights of GT heads, each split into three 16-bit numbers that add up to it: columns
// y * STRIDE + i, so that an mma that has eight columns anyway multiplies weights of 24 (bf16) or 33 bits (fp16) with the
// values at no cost.  Four heads have two columns each: a second mma (set) adds their third pieces.  Its first column of a head is no
// zero but the other half of the first piece, which makes that column the product with the first piece alone; see split_pieces.
// Two pieces (16 bits in bf16) were enough for a result of 8 bits unless it is a small difference of large terms.
// Against FMAs on unpacked values (8 conversions and 4 packed FMAs for 8 elements and head) this takes a half of the
// instructions for one head, a fifth for four.
template <int GT> struct Pieces {
    static constexpr int PIECES = 3, SETS = GT == 4 ? 2 : 1, STRIDE = 8 / (GT == 1 ? 2 : GT);
    // Piece in column STRIDE * y + i of a set, i < WIDTH.
    static constexpr int WIDTH = SETS == 2 ? 2 : PIECES;
    static __device__ __forceinline__ int piece_of(int set, int i) { return set == 1 && i == 1 ? 2 : i; }
    // Products with a first piece and with the others.  The first has the weight's sign, so that an infinite value times it is what it is times the
    // weight; the others may be zero or of the other sign, which makes NaN of it.  So where the first product is not finite it stands alone.
    // The sums of eight elements over a head's columns from the accumulators of lane t (acc[j][0], [1] and [2], [3]: elements j and j + 4 in
    // two columns).  STRIDE 2: those are all, h has the eight sums.  STRIDE 4: two lanes have a head, the first and second pieces and the
    // third and nothing, and each gets the sums of four elements, the even lane those of the first four.
    static constexpr int SUMS = STRIDE == 4 ? 4 : 8;
    static __device__ __forceinline__ void sum_columns(float (&h)[SUMS], const float (&acc)[4][4], int t) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float a = acc[j & 3][j / 4 * 2], b = acc[j & 3][j / 4 * 2 + 1];
            f[j] = a;
            if (fabsf(a) < INFINITY && !(STRIDE == 4 && (t & 1))) f[j] += b;
        }
#pragma unroll
        for (int e = 0; e < SUMS; ++e) {
            if constexpr (STRIDE == 4) {
                const float give = t & 1 ? f[e] : f[e + 4], keep = t & 1 ? f[e + 4] : f[e], got = __shfl_xor_sync(0xffffffffu, give, 1);
                const float sum = keep + got;                    // NaN also where the first pieces' is infinite and the third's of no use
                h[e] = sum == sum ? sum : t & 1 ? got : keep;
            } else {
                h[e] = f[e];
            }
        }
    }
};
template <typename T, int DMAX> struct ValueTile {
    static constexpr int CHUNKS = DMAX / 64;
    static __device__ __forceinline__ int element(int c, int g) { return CHUNKS == 1 ? g * 8 : c / 2 * 128 + g * 16 + c % 2 * 8; }
    uint4 r[4][CHUNKS];

    __device__ __forceinline__ void load(const T* pool, long base, int live, int D, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const T* first = pool + base;
        if (base >= 0 && live >= KEYS && D == DMAX && aligned32(first)) {
            const T* row = first + 2 * t * DMAX + element(0, g);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const T* at = row + ((i & 1) + (i >> 1) * 8) * DMAX;
                if constexpr (CHUNKS == 1) {
                    r[i][0] = load_once(at);
                } else {
#pragma unroll
                    for (int c = 0; c < CHUNKS; c += 2) load_once(at + c * 64, r[i][c], r[i][c + 1]);
                }
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = 2 * t + (i & 1) + (i >> 1) * 8;
            const bool on = base >= 0 && key < live;
            const T* row = pool + (on ? base + (long)key * D : 0);
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c) {
                const int e = element(c, g);
                r[i][c] = make_uint4(0, 0, 0, 0);
                if (on && e < D) r[i][c] = load_once((row + e));
            }
        }
    }
    // acc[c][j] += values x weights: [0], [1] element(c, g) + j, columns 2t and 2t + 1; [2], [3] element(c, g) + j + 4.
    template <int SETS> __device__ __forceinline__ void multiply(float (&acc)[CHUNKS][4][4], const uint32_t (&b)[SETS][2]) const {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t sel = j & 1 ? 0x7632 : 0x5410;
                const uint32_t lo[4] = {j < 2 ? r[0][c].x : r[0][c].y, j < 2 ? r[1][c].x : r[1][c].y, j < 2 ? r[2][c].x : r[2][c].y, j < 2 ? r[3][c].x : r[3][c].y};
                const uint32_t hi[4] = {j < 2 ? r[0][c].z : r[0][c].w, j < 2 ? r[1][c].z : r[1][c].w, j < 2 ? r[2][c].z : r[2][c].w, j < 2 ? r[3][c].z : r[3][c].w};
                const uint32_t a[4] = {__byte_perm(lo[0], lo[1], sel), __byte_perm(hi[0], hi[1], sel), __byte_perm(lo[2], lo[3], sel), __byte_perm(hi[2], hi[3], sel)};
#pragma unroll
                for (int s = 0; s < SETS; ++s) mma_16816<T>(acc[c][j], a[0], a[1], a[2], a[3], b[s][0], b[s][1]);
            }
        }
    }
};
// x as a sum of three numbers of type T; with two sets the first, which both have, counts twice.
template <typename T, int SETS> __device__ __forceinline__ void split_pieces(float x, float (&piece)[3]) {
    piece[0] = round_to<T>(SETS == 2 ? 0.5f * x : x);
    x = fmaf(-(float)SETS, piece[0], x);
    piece[1] = round_to<T>(x);
    piece[2] = round_to<T>(x - piece[1]);
}

// 2^x to a relative 2^-22; 0 below the smallest normal number.
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Work on sequences of different lengths is cut into `workers` equal runs of tiles; a run may begin in one sequence (line) and end
// in another.  Tile range of worker w of n tiles, and the worker that has tile x.
__device__ __forceinline__ long run_begin(long w, long n, long workers) { return w * n / workers; }
__device__ __forceinline__ long run_owner(long x, long n, long workers) { return ((x + 1) * workers - 1) / n; }

// before[b] = tiles of `1 << shift` keys in sequences 0..b-1, for b up to and with B; by the first warp of the block.
__device__ __forceinline__ void count_tiles(const PagedCache& c, int B, int shift, int* before, int* lens) {
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int sum = 0;
        for (int b0 = 0; b0 < B; b0 += 32) {
            const int len = b0 + lane < B ? c.length(b0 + lane) : 0;
            int n = (len + (1 << shift) - 1) >> shift;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, n, o);
                if (lane >= o) n += up;
            }
            if (b0 + lane < B) {
                before[b0 + lane + 1] = sum + n;
                lens[b0 + lane] = len;
            }
            sum += __shfl_sync(0xffffffffu, n, 31);
        }
        if (lane == 0) before[0] = 0;
    }
}

// Named barriers between warps of a block that hand work on: `n` threads, those that arrive and those that wait.  Both order the memory
// accesses before them.  Every call is reached by whole warps; the two sides count the same stages, so that every wait ends.
__device__ __forceinline__ void barrier_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void barrier_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }

// The last index b with before[b] <= x, x < before[B].
__device__ __forceinline__ int find_line(const int* before, int B, long x) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

// SMs of a B200.  The cuts of the work follow from the call's sizes alone, so that a workspace's size can be asked for without a device.
constexpr int DECODE_SMS = 148;
constexpr int DECODE_MAX_BATCH = 1024;   // batch rows of one call: their tile counts stand in shared memory
constexpr int DECODE_MAX_TAPS = 33;      // key taps: a tile's neighbours hold what its conv reaches
constexpr int DECODE_MAX_ROWS = 32;      // query rows that one new token looks at

// Launchers (paged_cache.cu, paged_conv_attn.cu, paged_mta.cu); abi_paged.cu has checked their arguments.  strides: elements between
// batch rows, heads and tokens of k, v and q.
int cache_append_launch(const PagedCache& cache, const void* k, const void* v, const void* q, const long* strides, const int* counts, int B, int T,
                        int dtype, cudaStream_t st);
int cache_copy_launch(void* k_pages, void* v_pages, const int* src, const int* dst, int n, long page_bytes, int pages, void* q_hist, const int* slot_src,
                      const int* slot_dst, int n_slots, long slot_bytes, int slots, int layers, cudaStream_t st);
size_t conv_attn_decode_workspace(int B, int H, int kv_heads, int D, int cq, int max_length);
int conv_attn_decode_launch(const PagedCache& cache, const void* w, int w_dtype, void* out, void* workspace, int B, int cq, int ck, float scale, int dtype,
                            cudaStream_t st);
// Fails where the heads' scores or probabilities do not fit in shared memory.
int mta_decode_workspace(int B, int H, int kv_heads, int D, int cq, int ck, int cq2, int ck2, int max_length, size_t* bytes);
int mta_decode_launch(const PagedCache& cache, const void* w1, const void* W1, const void* w2, const void* W2, int w_dtype, void* out, void* workspace, int B,
                      int cq, int ck, int cq2, int ck2, int dtype, cudaStream_t st);

}  // namespace mta
