// Conv attention of one new token per sequence over a paged cache:
//
//   s[i,k] = q[t-cq+1+i] . k[k] for k <= t-cq+1+i, else 0      (the last cq queries; t is the newest token)
//   c[k]   = sum_{i,j} w[h,i,j] s[i, k+j-(ck-1)/2]             k <= t
//   out    = sum_k softmax_k(scale * c[k]) v[k]
//
// Every key and value of a head is read once, for cq <= 8 about 2 D cq + 2 cq ck + 2 D = 1.9 kflop per 512 bytes at 6x11 taps and
// D 128: HBM bounds it, and what matters is that enough loads are in flight at every moment.  So a warp works alone, with no
// block-wide barrier: it walks a run of tiles of 16 keys; the scores of a tile are mma.sync chains (queries are the rows, keys the
// columns) into a ring of three tiles in shared memory, the conv of the tile before it reads that ring, its sixteen logits
// enter a running softmax (maximum, sum and output in float32 registers), and the loads of the next keys and values are issued
// as soon as the registers of the last ones are free.  Query heads that share keys are taken up to four at a time, side by side in the
// lanes.  Runs are equal cuts of all tiles of all sequences and heads, so lengths need not be alike; a second kernel joins the
// runs of a head.
//
// Measured (a graph of calls): one sequence of 131072 tokens, 16 heads, bf16, D 128 184 us, 5.8 TB/s; 32 of 1024 to 4096 tokens, fp16,
// D 64, 11x15 taps 102 us, 3.3 TB/s (conv and softmax chains of a warp: without the conv 79 us); 8 of 2048 to 8192 tokens, 32 heads on 8 key-value
// heads 75 us, 2.3 TB/s (instructions: four heads' convs per key); one of 517 tokens 11 us.
#include <type_traits>

#include "paged.cuh"

namespace mta {
namespace {

constexpr int WARPS = 4;
// Scores stand in pairs of query rows, (row 2i, row 2i + 1) side by side, so that one packed FMA serves two tap rows.
constexpr int RING = 3 * KEYS, RING_PITCH = 2 * RING + 8;   // floats of a pair of rows; the pitch spreads an accumulator's rows over the banks
constexpr int P_PITCH = KEYS + 8;                           // 16-bit weights of one column of the product with the values
constexpr float FP16_WEIGHT = 16384.0f;                     // scales weights, at most 1, so that what fp16's smallest number leaves of a piece is 2^-39

struct ConvAttnArgs {
    const void* w;
    void* out;
    float* part_o;         // (runs' parts, GT, D)
    float2* part_ml;       // (runs' parts, GT): maximum and sum
    int w_dtype, B, cq, ck;
    float scale;           // softmax scale * log2(e): the softmax runs in base 2
    int workers;
};

// Workers that have tiles when there are n tiles.  Runs of one tile read two more beside it, but of runs of four at least 517 tokens took
// 17 us instead of 11.
__device__ __forceinline__ long workers_of(const ConvAttnArgs& a, long n) { return n < a.workers ? n : a.workers; }

// Key taps are padded with zeros to a multiple of four; in shared memory 16 bytes more, so that the rows that lanes read at once lie in
// different banks.
__host__ __device__ constexpr int taps_padded(int ck) { return (ck + 3) / 4 * 4; }
__host__ __device__ constexpr int taps_pitch(int ck) { return taps_padded(ck) + 2; }

// Blocks that share an SM, by the bytes of a row: what the registers of a tile of keys, one of values and the outputs allow.  One block
// more at 256 bytes spilled 76 bytes a thread.
__host__ __device__ constexpr int blocks_per_sm(int row_bytes) { return row_bytes > 256 ? 2 : row_bytes > 128 ? 3 : 4; }

// Queries in shared memory.  16 bits: as the A operands of the scores' mma, [16 rows][half of a chunk][lane] 16 bytes, a conflict-free load
// each.  float32: rows, 64 bytes more than a multiple of 128 apart.
template <typename T, int DMAX, int NT> constexpr int query_bytes = sizeof(T) == 2 ? (NT + 1) / 2 * (DMAX * 2 / 32) * 512 : NT * 8 * (DMAX * 4 + 64);

// GT query heads that share a kv head, each with cq rows rounded up to pairs; NT * 8 >= all their rows of scores.
template <typename T, int DMAX, int GT, int NT> __host__ __device__ constexpr size_t conv_attn_warp_smem(int cq, int ck) {
    return (size_t)query_bytes<T, DMAX, NT> + (size_t)NT * 4 * RING_PITCH * 4 + (size_t)GT * ((cq + 1) / 2) * taps_pitch(ck) * 8 +
           (sizeof(T) == 2 ? Pieces<GT>::SETS * 8 * P_PITCH * 2 : GT * KEYS * 4);
}

// Two neighbouring keys of the conv, summed over the pairs of tap rows i, i + every, ...: .x the first rows of the pairs, .y the second.
// `first`: where the window begins in the ring, in units of two keys.  QUADS: taps / 4, 0: not known.
template <int QUADS> __device__ __forceinline__ void conv_row_pairs(float2& z0, float2& z1, const float* rows, const float* taps, int first, int i, int every, int cqp, int ckp) {
    const int steps = QUADS ? 2 * QUADS : ckp / 2;
    for (; i < cqp; i += every) {
        const float4 *srow = reinterpret_cast<const float4*>(rows + i * RING_PITCH), *wrow = reinterpret_cast<const float4*>(taps + i * (ckp + 2) * 2);
        int at = first;
        float4 lo = srow[at];
#pragma unroll
        for (int j = 0; j < steps; ++j) {
            at = at + 1 == RING / 2 ? 0 : at + 1;
            const float4 hi = srow[at], w = wrow[j];
            z0 = __ffma2_rn(make_float2(w.x, w.y), make_float2(lo.x, lo.y), z0);
            z1 = __ffma2_rn(make_float2(w.x, w.y), make_float2(lo.z, lo.w), z1);
            z0 = __ffma2_rn(make_float2(w.z, w.w), make_float2(lo.z, lo.w), z0);
            z1 = __ffma2_rn(make_float2(w.z, w.w), make_float2(hi.x, hi.y), z1);
            lo = hi;
        }
    }
}

template <typename T, int DMAX, int GT, int NT>
__global__ void __launch_bounds__(WARPS * 32, blocks_per_sm((int)sizeof(T) * DMAX)) conv_attn_decode_kernel(PagedCache c, ConvAttnArgs a) {
    constexpr bool HALF = sizeof(T) == 2;
    using K = KeyTile<T, DMAX>;
    using V = std::conditional_t<HALF, ValueTile<T, DMAX>, ValueTileF32<DMAX>>;
    using P = Pieces<GT>;
    constexpr int EPL = K::EPL;
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int cqp = (a.cq + 1) / 2, ckp = taps_padded(a.ck);
    char* mine = smem + warp * conv_attn_warp_smem<T, DMAX, GT, NT>(a.cq, a.ck);
    constexpr int QP = DMAX * (int)sizeof(T) + 64, QROWS = HALF ? (NT + 1) / 2 * 16 : NT * 8;
    char* q_sm = mine;
    float* s_sm = reinterpret_cast<float*>(mine + query_bytes<T, DMAX, NT>);
    float2* w_sm = reinterpret_cast<float2*>(s_sm + NT * 4 * RING_PITCH);       // [head][pair of tap rows][key tap]
    T* p_sm = reinterpret_cast<T*>(w_sm + GT * cqp * taps_pitch(a.ck));                      // [set][column][key]; float32: [head][key]
    int* before = reinterpret_cast<int*>(smem + WARPS * conv_attn_warp_smem<T, DMAX, GT, NT>(a.cq, a.ck));
    int* lens = before + a.B + 1;

    pdl_wait();
    count_tiles(c, a.B, 4, before, lens);
    __syncthreads();
    const int group = c.H / c.kv_heads, lines = c.H / GT;            // lines of one sequence: kv head, then GT query heads of it
    const long n = (long)before[a.B] * lines;
    const long workers = workers_of(a, n), me = (long)blockIdx.x * WARPS + warp;
    if (me >= workers) return;
    const long end = run_begin(me + 1, n, workers);
    const T* k_pool = static_cast<const T*>(c.k);
    const T* v_pool = static_cast<const T*>(c.v);
    const int left = (a.ck - 1) / 2, shift = left & 1;               // `shift` puts the window of an even key on a 16-byte boundary

    for (long x = run_begin(me, n, workers); x < end;) {
        int b = 0;
        {
            int lo = 0, hi = a.B;                                    // the sequence: last b with before[b] * lines <= x
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if ((long)before[mid] * lines <= x) lo = mid; else hi = mid;
            }
            b = lo;
        }
        const int len = lens[b], tiles = (len + KEYS - 1) / KEYS, slot = c.slot(b);
        const long in = x - (long)before[b] * lines;
        const int line = (int)(in / tiles), u0 = (int)(in - (long)line * tiles);
        const int u1 = (int)(end - x < tiles - u0 ? u0 + (end - x) : tiles);
        const int h0 = line * GT, kv_head = h0 / group;

        K keys;
        V values;
        auto live = [&](int u) { const int r = len - u * KEYS; return r < KEYS ? r : KEYS; };
        auto place = [&](int u) { return u >= 0 && u < tiles ? c.at(slot, kv_head, u * KEYS) : -1L; };
        long next = place(u0);                                       // of the keys to be loaded next; a tile's values lie where its keys do
        keys.load(k_pool, place(u0 - 1), KEYS, c.D, lane);           // a tile before this one is whole
        values.load(v_pool, next, live(u0), c.D, lane);
        long before_next = -1, values_at = -1;

        // queries and taps of this line
        for (int i = lane; i < QROWS * (DMAX / EPL); i += 32) {
            const int row = i / (DMAX / EPL), piece = i % (DMAX / EPL), e = piece * EPL, gq = row / (2 * cqp), tap = row % (2 * cqp), pos = len - a.cq + tap;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (gq < GT && tap < a.cq && pos >= 0 && e < c.D)
                u = *reinterpret_cast<const uint4*>(static_cast<const T*>(c.q_hist) + (((long)slot * c.ring + pos % c.ring) * c.H + h0 + gq) * c.D + e);
            if constexpr (HALF) {
                // 16 bytes of a row: the first two registers of one half of the chunk, then of the other, for lane (row % 8, position)
                // 16 bytes number `piece` of a row are chunk 2p + piece % 2, p = piece / 8, of position piece / 2 % 4
                uint32_t* to = reinterpret_cast<uint32_t*>(q_sm + ((row / 16 * K::CH + piece / 8 * 2 + piece % 2) * 2 * 32 + row % 8 * 4 + piece / 2 % 4) * 16) + row / 8 % 2;
                to[0] = u.x; to[2] = u.y; to[128] = u.z; to[130] = u.w;
            } else {
                *reinterpret_cast<uint4*>(q_sm + row * QP + e * (int)sizeof(T)) = u;
            }
        }
        for (int i = lane; i < GT * cqp * ckp; i += 32) {
            const int j = i % ckp, pair = i / ckp % cqp, y = i / ckp / cqp;
            const long at = ((long)(h0 + y) * a.cq + 2 * pair) * a.ck + j;
            w_sm[i / ckp * taps_pitch(a.ck) + j] = make_float2(j < a.ck ? load_weight(a.w, at, a.w_dtype) * a.scale : 0.0f,
                                  j < a.ck && 2 * pair + 1 < a.cq ? load_weight(a.w, at + a.ck, a.w_dtype) * a.scale : 0.0f);
        }
        if constexpr (HALF) {
            for (int i = lane; i < P::SETS * 8 * P_PITCH / 2; i += 32) reinterpret_cast<uint32_t*>(p_sm)[i] = 0;      // columns that no piece fills
        }
        __syncwarp();

        // lane (head, share of the tap rows, pair of keys): maximum of its head, sum of its own keys
        constexpr int SHARES = 4 / GT;
        const int my_head = lane / (8 * SHARES), share = (lane >> 3) % SHARES, pair = lane & 7;
        float m = -INFINITY, l = 0.0f;
        float o[HALF ? DMAX / 64 : GT][4][4];                        // mma accumulators; float32: [head][0][element]
#pragma unroll
        for (int i = 0; i < (HALF ? DMAX / 64 : GT); ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;

        for (int u = u0 - 1; u <= u1; ++u) {
            constexpr int PARTS = K::template PARTS<NT * 8>;
            float acc[PARTS][4];
            keys.template score<NT * 8>(acc, lane, [&](int row, int ch) {
                if constexpr (HALF) return reinterpret_cast<const uint4*>(q_sm)[(row * 2 * K::CH + ch) * 32 + lane];
                else return *reinterpret_cast<const uint4*>(q_sm + row * QP + K::element(ch, t4) * 4);
            });
            if (u < u1) {
                keys.load(k_pool, next, live(u + 1), c.D, lane);
                const long loaded = next;
                next = place(u + 2);                                 // looked up an iteration before it is used
                values_at = before_next;
                before_next = loaded;
            }
            const int col = ((u + 3) % 3) * KEYS + shift;
            // scores above the diagonal are zero; those of tiles outside the sequence are zero already
            if (u * KEYS + KEYS - 1 > len - a.cq) {
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (u * KEYS + K::key_of(p, i, lane) > len - a.cq + K::row_of(p, i, lane) % (2 * cqp)) acc[p][i] = 0.0f;
            }
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = K::row_of(p, i, lane);
                    int at = col + K::key_of(p, i, lane);
                    if (at >= RING) at -= RING;
                    if (row < NT * 8) s_sm[(row >> 1) * RING_PITCH + 2 * at + (row & 1)] = acc[p][i];
                }
            }
            __syncwarp();
            if (u > u0) {
                const int un = u - 1;
                int first = (un % 3) * KEYS + 2 * pair + shift - left;             // even
                if (first < 0) first += RING;
                float2 z0 = make_float2(0.0f, 0.0f), z1 = z0;
                const float *rows = s_sm + my_head * cqp * RING_PITCH, *taps = reinterpret_cast<const float*>(w_sm + my_head * cqp * taps_pitch(a.ck));
                switch (ckp / 4) {
                    case 1: conv_row_pairs<1>(z0, z1, rows, taps, first / 2, share, SHARES, cqp, ckp); break;
                    case 2: conv_row_pairs<2>(z0, z1, rows, taps, first / 2, share, SHARES, cqp, ckp); break;
                    case 3: conv_row_pairs<3>(z0, z1, rows, taps, first / 2, share, SHARES, cqp, ckp); break;
                    case 4: conv_row_pairs<4>(z0, z1, rows, taps, first / 2, share, SHARES, cqp, ckp); break;
                    default: conv_row_pairs<0>(z0, z1, rows, taps, first / 2, share, SHARES, cqp, ckp); break;
                }
                float z[2] = {z0.x + z0.y, z1.x + z1.y}, p[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int s = 8; s < 8 * SHARES; s <<= 1) z[e] += __shfl_xor_sync(0xffffffffu, z[e], s);
                    if (un * KEYS + 2 * pair + e >= len) z[e] = -INFINITY;
                }
                float top = fmaxf(z[0], z[1]);
#pragma unroll
                for (int s = 1; s < 8; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                top = fmaxf(m, top);
                // while every logit so far is -inf nothing has been summed: a finite stand-in keeps -inf - -inf away
                const float ref = top == -INFINITY ? 0.0f : top, fade = fast_exp2(m - ref);
                const bool moved = __any_sync(0xffffffffu, top != m);
                m = top;
                p[0] = fast_exp2(z[0] - ref);
                p[1] = fast_exp2(z[1] - ref);
                l = fmaf(l, fade, p[0] + p[1]);
                if constexpr (HALF) {
                    constexpr float by = std::is_same_v<T, __half> ? FP16_WEIGHT : 1.0f;
                    float a0[P::PIECES], a1[P::PIECES];
                    split_pieces<T, P::SETS>(p[0] * by, a0);
                    split_pieces<T, P::SETS>(p[1] * by, a1);
                    // the lanes that hold these keys share the pieces out
#pragma unroll
                    for (int s = 0; s < P::SETS; ++s)
#pragma unroll
                        for (int i = 0; i < P::WIDTH; ++i)
                            if (i % SHARES == share)
                                *reinterpret_cast<uint32_t*>(p_sm + (s * 8 + my_head * P::STRIDE + i) * P_PITCH + 2 * pair) = pack2<T>(a0[P::piece_of(s, i)], a1[P::piece_of(s, i)]);
                } else {
                    if (share == 0) *reinterpret_cast<float2*>(p_sm + my_head * KEYS + 2 * pair) = make_float2(p[0], p[1]);
                }
                __syncwarp();
                if constexpr (HALF) {
                    if (moved) {
                        // the head of this lane's two columns
                        const int y = 2 * t4 / P::STRIDE;
                        const float f = __shfl_sync(0xffffffffu, fade, (y < GT ? y : 0) * 8 * SHARES);
#pragma unroll
                        for (int i = 0; i < V::CHUNKS; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) { o[i][j][0] *= f; o[i][j][1] *= f; o[i][j][2] *= f; o[i][j][3] *= f; }
                    }
                    uint32_t w[P::SETS][2];
#pragma unroll
                    for (int s = 0; s < P::SETS; ++s) {
                        const uint32_t* col_p = reinterpret_cast<const uint32_t*>(p_sm + (s * 8 + g) * P_PITCH) + t4;
                        w[s][0] = col_p[0];
                        w[s][1] = col_p[4];
                    }
                    values.multiply(o, w);
                } else {
#pragma unroll
                    for (int y = 0; y < GT; ++y) {
                        const float f = __shfl_sync(0xffffffffu, fade, y * 8 * SHARES);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[y][0][e] *= f;
                    }
#pragma unroll
                    for (int i = 0; i < V::STEPS; ++i) {
                        float f[4];
                        unpack16(values.r[i], f);
#pragma unroll
                        for (int y = 0; y < GT; ++y) {
                            const float p = p_sm[y * KEYS + i * V::SUBS + lane / V::ROWLANES];
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[y][0][e] = fmaf(p, f[e], o[y][0][e]);
                        }
                    }
                }
                if (u < u1) values.load(v_pool, values_at, live(u), c.D, lane);
            }
            __syncwarp();
        }
        const bool all = u0 == 0 && u1 == tiles;                     // the whole line: nothing to join
        const long part = me + (long)b * lines + line;
#pragma unroll
        for (int s = 1; s < 8; s <<= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
        float sums[GT];
#pragma unroll
        for (int y = 0; y < GT; ++y) sums[y] = __shfl_sync(0xffffffffu, l, y * 8 * SHARES);
        if (lane % (8 * SHARES) == 0 && !all) a.part_ml[part * GT + my_head] = make_float2(m, l);
        // Stores four elements of head y from element e0 on.
        auto store = [&](int y, int e0, const float* f) {
            if (all) {
                T* to = static_cast<T*>(a.out) + ((long)b * c.H + h0 + y) * c.D + e0;
                const float r[4] = {f[0] / sums[y], f[1] / sums[y], f[2] / sums[y], f[3] / sums[y]};
                if constexpr (HALF) *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(r[0], r[1]), pack2<T>(r[2], r[3]));
                else *reinterpret_cast<float4*>(to) = make_float4(r[0], r[1], r[2], r[3]);
            } else {
                *reinterpret_cast<float4*>(a.part_o + (part * GT + y) * c.D + e0) = make_float4(f[0], f[1], f[2], f[3]);
            }
        };
        if constexpr (HALF) {
            constexpr float by = std::is_same_v<T, __half> ? 1.0f / FP16_WEIGHT : 1.0f;
#pragma unroll
            for (int i = 0; i < V::CHUNKS; ++i) {
                float f[P::SUMS];
                P::sum_columns(f, o[i], t4);
#pragma unroll
                for (int e = 0; e < P::SUMS; ++e) f[e] *= by;
                const int e0 = V::element(i, g);
#pragma unroll
                for (int y = 0; y < GT; ++y) {
                    if (t4 * 2 / P::STRIDE != y || e0 >= c.D) continue;
                    if constexpr (P::STRIDE == 4) {
                        store(y, e0 + (t4 & 1) * 4, f);
                    } else {
                        store(y, e0, f);
                        store(y, e0 + 4, f + 4);
                    }
                }
            }
        } else {
#pragma unroll
            for (int y = 0; y < GT; ++y) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int s = V::ROWLANES; s < 32; s <<= 1) o[y][0][e] += __shfl_xor_sync(0xffffffffu, o[y][0][e], s);
                if (lane < V::ROWLANES && lane * 4 < c.D) store(y, lane * 4, o[y][0]);
            }
        }
        x += u1 - u0;
        __syncwarp();
    }
}

// One block per (head, sequence): the parts of its runs, in the order of their keys.  Sequences of no tokens get zeros.
template <typename T> __global__ void __launch_bounds__(128) conv_attn_join_kernel(PagedCache c, ConvAttnArgs a, int GT) {
    extern __shared__ __align__(16) char smem[];
    int* before = reinterpret_cast<int*>(smem);
    int* lens = before + a.B + 1;
    __shared__ float sum_l[4];
    __shared__ float sum_o[4][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.x, b = blockIdx.y;
    count_tiles(c, a.B, 4, before, lens);
    __syncthreads();
    pdl_wait();
    T* out = static_cast<T*>(a.out) + ((long)b * c.H + h) * c.D;
    const int tiles = before[b + 1] - before[b];
    if (tiles == 0) {
        for (int d = threadIdx.x; d < c.D; d += 128) out[d] = from_f32<T>(0.0f);
        return;
    }
    const int lines = c.H / GT, line = h / GT, y = h % GT;
    const long n = (long)before[a.B] * lines, workers = workers_of(a, n);
    const long x = (long)before[b] * lines + (long)line * tiles;
    const long w0 = run_owner(x, n, workers), w1 = run_owner(x + tiles - 1, n, workers);
    if (w0 == w1) return;                                            // that run wrote the result
    const long part0 = w0 + (long)b * lines + line;
    const int parts = (int)(w1 - w0) + 1;
    float top = -INFINITY;
    for (int p = lane; p < parts; p += 32) top = fmaxf(top, a.part_ml[(part0 + p) * GT + y].x);
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    float l = 0.0f;
    float4 o[2] = {make_float4(0, 0, 0, 0), make_float4(0, 0, 0, 0)};
#pragma unroll 4
    for (int p = warp; p < parts; p += 4) {
        const float2 ml = a.part_ml[(part0 + p) * GT + y];
        const float f = exp2f(ml.x - top);
        l += ml.y * f;
        const float4* from = reinterpret_cast<const float4*>(a.part_o + ((part0 + p) * GT + y) * c.D);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if ((lane + 32 * i) * 4 < c.D) {
                const float4 v = from[lane + 32 * i];
                o[i].x = fmaf(v.x, f, o[i].x); o[i].y = fmaf(v.y, f, o[i].y); o[i].z = fmaf(v.z, f, o[i].z); o[i].w = fmaf(v.w, f, o[i].w);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if ((lane + 32 * i) * 4 < c.D) *reinterpret_cast<float4*>(&sum_o[warp][(lane + 32 * i) * 4]) = o[i];
    if (lane == 0) sum_l[warp] = l;
    __syncthreads();
    l = sum_l[0] + sum_l[1] + sum_l[2] + sum_l[3];
    for (int d = threadIdx.x; d < c.D; d += 128) out[d] = from_f32<T>((sum_o[0][d] + sum_o[1][d] + sum_o[2][d] + sum_o[3][d]) / l);
}

// Query heads that a warp takes together: up to four that share a kv head, if their scores, an even number of rows each, fit in 32 rows.
int heads_together(int group, int cq) {
    const int rows = (cq + 1) / 2 * 2;
    if (group % 4 == 0 && 4 * rows <= DECODE_MAX_ROWS) return 4;
    if (group % 2 == 0 && 2 * rows <= DECODE_MAX_ROWS) return 2;
    return 1;
}

struct Plan {
    int gt, workers;
    size_t ml_bytes, bytes;
};

// Room for as many runs as there can be for any type; `row_bytes` (0: not known) sets the number of this call's.
Plan make_plan(int B, int H, int kv_heads, int D, int cq, int max_length, int row_bytes) {
    Plan plan, *p = &plan;
    p->gt = heads_together(H / kv_heads, cq);
    const long lines = (long)B * (H / p->gt), tiles = lines * ((max_length + KEYS - 1) / KEYS);
    long workers = tiles;
    const long most = (long)DECODE_SMS * WARPS * blocks_per_sm(0);
    if (workers > most) workers = most;
    if (workers < 1) workers = 1;
    const size_t parts = (size_t)(workers + lines) * p->gt;
    p->ml_bytes = (parts * sizeof(float2) + 255) / 256 * 256;
    p->bytes = p->ml_bytes + parts * D * sizeof(float);
    const long wave = (long)DECODE_SMS * WARPS * blocks_per_sm(row_bytes);
    p->workers = (int)(workers < wave ? workers : wave);
    return plan;
}

template <typename T, int DMAX, int GT, int NT>
int launch(const PagedCache& c, const ConvAttnArgs& a, cudaStream_t st) {
    const size_t smem = WARPS * conv_attn_warp_smem<T, DMAX, GT, NT>(a.cq, a.ck) + (2 * a.B + 1) * sizeof(int);
    if (int rc = launch_kernel<conv_attn_decode_kernel<T, DMAX, GT, NT>>("conv_attn_decode_kernel", dim3((a.workers + WARPS - 1) / WARPS), WARPS * 32, smem, st, c, a))
        return rc;
    return launch_kernel<conv_attn_join_kernel<T>>("conv_attn_join_kernel", dim3(c.H, a.B), 128, (2 * a.B + 1) * sizeof(int), st, c, a, GT);
}

template <typename T, int DMAX> int launch_rows(const PagedCache& c, const ConvAttnArgs& a, int gt, cudaStream_t st) {
    const int nt = (gt * ((a.cq + 1) / 2 * 2) + 7) / 8;
    if (gt == 4) return nt <= 3 ? launch<T, DMAX, 4, 3>(c, a, st) : launch<T, DMAX, 4, 4>(c, a, st);
    if (gt == 2) return nt <= 2 ? launch<T, DMAX, 2, 2>(c, a, st) : launch<T, DMAX, 2, 4>(c, a, st);
    return nt <= 1 ? launch<T, DMAX, 1, 1>(c, a, st) : nt <= 2 ? launch<T, DMAX, 1, 2>(c, a, st) : launch<T, DMAX, 1, 4>(c, a, st);
}

template <typename T> int launch_dim(const PagedCache& c, const ConvAttnArgs& a, int gt, cudaStream_t st) {
    if (c.D <= 64) return launch_rows<T, 64>(c, a, gt, st);
    if constexpr (sizeof(T) == 4) return launch_rows<T, 128>(c, a, gt, st);
    else return c.D <= 128 ? launch_rows<T, 128>(c, a, gt, st) : launch_rows<T, 256>(c, a, gt, st);
}

}  // namespace

size_t conv_attn_decode_workspace(int B, int H, int kv_heads, int D, int cq, int max_length) {
    return make_plan(B, H, kv_heads, D, cq, max_length, 0).bytes;
}

int conv_attn_decode_launch(const PagedCache& cache, const void* w, int w_dtype, void* out, void* workspace, int B, int cq, int ck, float scale, int dtype,
                            cudaStream_t st) {
    PagedCache c = cache;
    if (int rc = wait_flag_ptr(&c.err)) return rc;
    const Plan p = make_plan(B, c.H, c.kv_heads, c.D, cq, c.max_length, (c.D <= 64 ? 64 : c.D <= 128 ? 128 : 256) * (int)dtype_size(dtype));
    ConvAttnArgs a;
    a.w = w; a.w_dtype = w_dtype; a.out = out; a.B = B; a.cq = cq; a.ck = ck; a.scale = scale * LOG2E;
    a.part_ml = static_cast<float2*>(workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.ml_bytes);
    a.workers = p.workers;
    if (dtype == MTA_F32) return launch_dim<float>(c, a, p.gt, st);
    return dtype == MTA_BF16 ? launch_dim<__nv_bfloat16>(c, a, p.gt, st) : launch_dim<__half>(c, a, p.gt, st);
}

}  // namespace mta
