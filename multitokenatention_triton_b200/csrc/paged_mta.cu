// The MTA module for one new token per sequence over a paged cache.  With t the newest token, R = cq + cq2 - 1 and pos(j) = t-R+1+j:
//
//   s[h,j,k] = scale * q[h,pos(j)] . k[h,k] for 0 <= k <= pos(j), else 0           j < R
//   c[h,r,k] = sum_{i,j} w1[h,i,j] s[h,r+i,k+j-(ck-1)/2]                           r < cq2
//   l[o,r,k] = sum_h W1[o,h] c[h,r,k];  p[o,r,.] = softmax over k <= pos(cq-1+r); a row before the first token has p = 0
//   y[h,k]   = sum_{i,j} w2[h,i,j] p[h,i,k+j-(ck2-1)/2],  k <= t
//   out[o]   = sum_k (sum_h W2[o,h] y[h,k]) v[o,k]
//
// The rows before the newest are computed again from the last R queries instead of being kept: with the queries as the eight
// columns of an mma they cost no byte more, and a cache that holds keys, values and R queries can be forked or moved at any token.
// Both head mixes need all heads of a key, the softmax all keys of a row, so the work is three kernels:
//   scores  block = a run of key tiles, all heads: scores, conv, head mix; logits to the workspace (float32, base 2),
//           maximum and sum of every (row, head) of the run
//   values  the same runs: joins the maxima and sums of all runs, probabilities, conv, head mix, product with the values
//   join    adds the runs' outputs
// Keys and values are read once; the logits add 4 cq2 bytes written and read, mostly in L2, to the 4 D of keys and values in 16 bits.
#include <type_traits>

#include "paged.cuh"

namespace mta {
namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32;

struct MtaArgs {
    const void *w1, *W1, *w2, *W2;
    void* out;
    float* logits;         // (B, cq2, H, pitch)
    float2* part_ml;       // (parts, cq2, H)
    float* part_o;         // (parts, H, D)
    long pitch;
    int w_dtype, B, cq, ck, cq2, ck2;
    float scale;           // log2(e) / sqrt(D), taken into the first conv's taps: logits are in base 2
    int workers, shift;    // key tiles of 1 << shift
    int kv_together;       // kv heads whose scores fit in shared memory at once
};

__host__ __device__ inline int round4(int x) { return (x + 3) / 4 * 4; }
__host__ __device__ inline int halo(int x) { return (x + KEYS - 1) / KEYS * KEYS; }

// The scores of a tile and its neighbours: a ring of `keys` positions, so that what two tiles share is computed once.  Two heads
// stand side by side, which lets one packed FMA serve both.  Keys (4i, 4i + 1) lie in the first half of a row, (4i + 2, 4i + 3) in
// the second, 16 bytes each: the conv's threads, four keys apart, read neighbouring 16 bytes.  The pads put the rows and halves that an
// accumulator writes at once into different banks.
struct ScoreRing {
    int keys, half, row;   // floats of half a row and of a row
    __host__ __device__ ScoreRing(int tile, int ck) {
        keys = halo((ck - 1) / 2) + tile + halo(ck - 1 - (ck - 1) / 2);
        half = keys + (keys % 32 == 0 ? 8 : 24);
        row = 2 * half + 8;
    }
};
__host__ __device__ inline int prob_pitch(int tile, int ck2) { return tile + round4(ck2) + 4; }

struct ScoreSmem {
    size_t s, c, W, taps, ml, q_at, before, bytes;
};
__host__ __device__ inline ScoreSmem score_smem(int B, int H, int group, int kv_together, int tile, int cq, int ck, int cq2) {
    ScoreSmem m;
    size_t at = 0;
    const int R = cq + cq2 - 1;
    m.s = at; at += (size_t)((kv_together * group + 1) / 2) * R * ScoreRing(tile, ck).row * 4;
    m.c = at; at += (size_t)cq2 * H * tile * 4;
    m.W = at; at += (size_t)H * round4(H) * 4;
    m.taps = at; at += (size_t)((H + 1) / 2) * cq * round4(ck) * 8;
    m.ml = at; at += ((size_t)cq2 * H * 8 + 15) / 16 * 16;
    m.q_at = at; at += DECODE_MAX_ROWS * 8;
    m.before = at; at += (size_t)(2 * B + 1) * 4;
    m.bytes = at;
    return m;
}
// 16-bit pieces of the weights in a row of `tile` keys; the pad spreads eight rows over the banks.
__host__ __device__ inline int piece_pitch(int tile) { return tile + 8; }
struct ValueSmem {
    size_t p, y, a, W, taps, ml, by, o, before, bytes;
};
__host__ __device__ inline ValueSmem value_smem(int B, int H, int D, int tile, int cq2, int ck2, int copies) {
    ValueSmem m;
    size_t at = 0;
    m.p = at; at += (size_t)cq2 * H * prob_pitch(tile, ck2) * 4;
    m.y = at; at += (size_t)H * tile * 4;
    m.a = at; at += (size_t)H * (3 * piece_pitch(tile) * 2);     // up to three pieces; float32: 4 bytes a key
    m.W = at; at += (size_t)H * round4(H) * 4;
    m.taps = at; at += (size_t)H * cq2 * round4(ck2) * 4;
    m.ml = at; at += ((size_t)cq2 * H * 8 + 15) / 16 * 16;
    m.by = at; at += (size_t)round4(H) * 4;
    m.o = at; at += (size_t)copies * H * D * 4;
    m.before = at; at += (size_t)(2 * B + 1) * 4;
    m.bytes = at;
    return m;
}

// W transposed to [h][o], so that four outputs are one 16-byte load.
__device__ __forceinline__ void load_mix(float* W, const void* from, int H, int w_dtype) {
    const int Hp = round4(H);
    for (int i = threadIdx.x; i < H * Hp; i += THREADS) {
        const int o = i / H, h = i - o * H;                      // neighbouring threads read neighbouring weights
        W[h * Hp + o] = o < H ? load_weight(from, (long)o * H + h, w_dtype) : 0.0f;
    }
}

// Four neighbouring outputs of a conv row: windows of `x` from its first element on (16-byte aligned), ckp taps.
__device__ __forceinline__ void conv_row(float (&z)[4], const float* x, const float* w, int ckp) {
    const float4 *xs = reinterpret_cast<const float4*>(x), *ws = reinterpret_cast<const float4*>(w);
    float4 lo = xs[0];
    for (int j = 0; j < ckp / 4; ++j) {
        const float4 hi = xs[j + 1], t = ws[j];
        z[0] = fmaf(t.x, lo.x, fmaf(t.y, lo.y, fmaf(t.z, lo.z, fmaf(t.w, lo.w, z[0]))));
        z[1] = fmaf(t.x, lo.y, fmaf(t.y, lo.z, fmaf(t.z, lo.w, fmaf(t.w, hi.x, z[1]))));
        z[2] = fmaf(t.x, lo.z, fmaf(t.y, lo.w, fmaf(t.z, hi.x, fmaf(t.w, hi.y, z[2]))));
        z[3] = fmaf(t.x, lo.w, fmaf(t.y, hi.x, fmaf(t.z, hi.y, fmaf(t.w, hi.z, z[3]))));
        lo = hi;
    }
}

// z[o][k] = sum_h W[h][o0 + o] from[h][k0 + k] for four heads and four keys.
__device__ __forceinline__ void mix_heads(float (&z)[4][4], const float* W, const float* from, int H, int tile) {
    const int Hp = round4(H);
#pragma unroll
    for (int o = 0; o < 4; ++o) z[o][0] = z[o][1] = z[o][2] = z[o][3] = 0.0f;
#pragma unroll 4
    for (int h = 0; h < H; ++h) {
        const float4 x = *reinterpret_cast<const float4*>(from + h * tile), w = *reinterpret_cast<const float4*>(W + h * Hp);
        const float ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            z[o][0] = fmaf(ws[o], x.x, z[o][0]); z[o][1] = fmaf(ws[o], x.y, z[o][1]);
            z[o][2] = fmaf(ws[o], x.z, z[o][2]); z[o][3] = fmaf(ws[o], x.w, z[o][3]);
        }
    }
}

// Asks L2 for the rows of `tile` keys of every kv head from key k0 on: 16 keys a thread.
template <typename T> __device__ __forceinline__ void prefetch_tile(const PagedCache& c, const T* pool, int slot, int k0, int tile, int len) {
    const int units = tile / KEYS;
    for (int i = threadIdx.x; i < c.kv_heads * units; i += THREADS) {
        const int key = k0 + i % units * KEYS;
        if (key >= len) continue;
        const long base = c.at(slot, i / units, key);
        if (base >= 0) prefetch_l2(pool + base, (uint32_t)((len - key < KEYS ? len - key : KEYS) * c.D * sizeof(T)));
    }
}

// Blocks an SM: one where two would spill registers (wide rows, many query rows, float32 with more than eight rows).
__host__ __device__ constexpr int scores_blocks(int elem, int dmax, int nt) { return elem * dmax > 256 || nt == 4 || (elem == 4 && nt > 1) ? 1 : 2; }

template <typename T, int DMAX, int NT>
__global__ void __launch_bounds__(THREADS, scores_blocks((int)sizeof(T), DMAX, NT)) mta_decode_scores_kernel(PagedCache c, MtaArgs a) {
    constexpr bool HALF = sizeof(T) == 2;
    using K = KeyTile<T, DMAX>;
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int H = c.H, group = H / c.kv_heads, tile = 1 << a.shift, R = a.cq + a.cq2 - 1, ckp = round4(a.ck);
    const int left = (a.ck - 1) / 2, hl = halo(left), hr = halo(a.ck - 1 - left);
    const int shift = left & 3;                                  // puts the windows of a tile's quads of keys on 16-byte boundaries
    const ScoreRing ring(tile, a.ck);
    const ScoreSmem m = score_smem(a.B, H, group, a.kv_together, tile, a.cq, a.ck, a.cq2);
    float *s_sm = reinterpret_cast<float*>(smem + m.s), *c_sm = reinterpret_cast<float*>(smem + m.c), *W_sm = reinterpret_cast<float*>(smem + m.W);
    float2 *t_sm = reinterpret_cast<float2*>(smem + m.taps), *ml = reinterpret_cast<float2*>(smem + m.ml);
    long* q_at = reinterpret_cast<long*>(smem + m.q_at);
    int *before = reinterpret_cast<int*>(smem + m.before), *lens = before + a.B + 1;

    pdl_wait();
    count_tiles(c, a.B, a.shift, before, lens);
    load_mix(W_sm, a.W1, H, a.w_dtype);
    for (int i = threadIdx.x; i < (H + 1) / 2 * a.cq * ckp; i += THREADS) {
        const int j = i % ckp, row = i / ckp, tap = row % a.cq, h = row / a.cq * 2;
        const long at = ((long)h * a.cq + tap) * a.ck + j;
        t_sm[i] = make_float2(j < a.ck ? load_weight(a.w1, at, a.w_dtype) * a.scale : 0.0f,
                              j < a.ck && h + 1 < H ? load_weight(a.w1, at + a.cq * a.ck, a.w_dtype) * a.scale : 0.0f);
    }
    // positions that hold no score yet are read with taps of zero: they have to be finite
    for (int i = threadIdx.x; i < (a.kv_together * group + 1) / 2 * R * ring.row / 4; i += THREADS) reinterpret_cast<float4*>(s_sm)[i] = make_float4(0, 0, 0, 0);
    __syncthreads();
    const long n = before[a.B], workers = n < a.workers ? n : a.workers, me = blockIdx.x;
    if (me >= workers) return;
    const long end = run_begin(me + 1, n, workers);
    const T* pool = static_cast<const T*>(c.k);
    const T* queries = static_cast<const T*>(c.q_hist);
    const bool whole = a.kv_together == c.kv_heads;              // all heads at once: what tiles share stays in the ring
    const int quads = tile / 4, oquads = round4(H) / 4;

    for (long x = run_begin(me, n, workers); x < end;) {
        const int b = find_line(before, a.B, x), len = lens[b], slot = c.slot(b);
        const int ta = (int)(x - before[b]), tb = (int)(end - before[b] < before[b + 1] - before[b] ? end - before[b] : before[b + 1] - before[b]);
        for (int i = threadIdx.x; i < a.cq2 * H; i += THREADS) ml[i] = make_float2(-INFINITY, 0.0f);
        if (threadIdx.x < DECODE_MAX_ROWS) {
            const int pos = len - R + threadIdx.x;
            q_at[threadIdx.x] = threadIdx.x < R && pos >= 0 ? ((long)slot * c.ring + pos % c.ring) * H * c.D : -1;
        }
        __syncthreads();
        for (int tl = ta; tl < tb; ++tl) {
            const int k0 = tl << a.shift;
            if (tl + 1 < tb) prefetch_tile(c, pool, slot, k0 + tile + hr, tile, len);
            for (int hk0 = 0; hk0 < c.kv_heads; hk0 += a.kv_together) {
                const int nk = c.kv_heads - hk0 < a.kv_together ? c.kv_heads - hk0 : a.kv_together;
                // scores of the keys that the ring does not hold yet, one (kv head, 16 keys) a warp and step
                const int first = whole && tl > ta ? k0 + hr : k0 - hl, units = (k0 + tile + hr - first) / KEYS, tasks = nk * units;
                K keys;
                uint4 q[HALF ? NT : 1][HALF ? K::CH : 1];
                auto fetch = [&](int hk, int key) {
                    keys.load(pool, key >= 0 && key < len ? c.at(slot, hk0 + hk, key) : -1L, len - key < KEYS ? len - key : KEYS, c.D, lane);
                };
                int task = warp * tasks / WARPS;
                const int last = (warp + 1) * tasks / WARPS;
                int hk = task / units, u = task - hk * units, q_head = -1;
                if (task < last) fetch(hk, first + u * KEYS);
                while (task < last) {
                    const int key = first + u * KEYS, hk_now = hk;
                    ++task;
                    if (++u == units) { u = 0; ++hk; }
                    int at = (key + shift + ring.keys) % ring.keys + g;              // ring position of key `g` of the unit
                    const bool full = key + KEYS - 1 <= len - R;                     // every row sees every key
                    for (int gq = 0; gq < group; ++gq) {
                        const int h = hk_now * group + gq;
                        const T* qh = queries + (long)(hk0 * group + h) * c.D;
                        float acc[NT][4];
                        if constexpr (HALF) {
                            if (q_head != h) {
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    const long row = q_at[8 * nt + g];
#pragma unroll
                                    for (int ch = 0; ch < K::CH; ++ch) {
                                        const int e = (ch * 4 + t4) * K::EPL;
                                        q[nt][ch] = row >= 0 && e < c.D ? *reinterpret_cast<const uint4*>(qh + row + e) : make_uint4(0, 0, 0, 0);
                                    }
                                }
                                q_head = h;
                            }
                            keys.template score<NT>(acc, lane, [&](int nt, int ch) { return q[nt][ch]; });
                        } else {
                            keys.template score<NT>(acc, lane, [&](int row, int ch) {
                                const long r = q_at[row];
                                const int e = (ch * 4 + t4) * K::EPL;
                                return r >= 0 && e < c.D ? *reinterpret_cast<const uint4*>(qh + r + e) : make_uint4(0, 0, 0, 0);
                            });
                        }
                        if (gq == group - 1 && task < last) fetch(hk, first + u * KEYS);
                        float* s = s_sm + (long)(h >> 1) * R * ring.row + (h & 1);
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            int pos = at + 8 * y;
                            if (pos >= ring.keys) pos -= ring.keys;
                            const int place = (pos & 2 ? ring.half : 0) + (pos >> 2) * 4 + (pos & 1) * 2, kk = key + g + 8 * y;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                                for (int z = 0; z < 2; ++z) {
                                    const int row = 8 * nt + 2 * t4 + z;
                                    if (row < R) s[row * ring.row + place] = full || kk <= len - R + row ? acc[nt][2 * y + z] : 0.0f;
                                }
                            }
                        }
                    }
                }
                __syncthreads();
                // conv: (two heads, row, four keys) a thread
                const int heads = nk * group, pairs = (heads + 1) / 2;
                int q0 = k0 - left + shift;                                          // a multiple of 4
                q0 = ((q0 + ring.keys) % ring.keys) >> 2;
                for (int i = threadIdx.x; i < pairs * a.cq2 << (a.shift - 2); i += THREADS) {
                    const int quad = i & (quads - 1), rest = i >> (a.shift - 2), r = rest / pairs, pair = rest - r * pairs;
                    int q1 = q0 + quad;
                    if (q1 >= ring.keys / 4) q1 -= ring.keys / 4;
                    float2 z[4];
                    z[0] = z[1] = z[2] = z[3] = make_float2(0.0f, 0.0f);
                    const float* srow = s_sm + ((long)pair * R + r) * ring.row;
                    const float4* w = reinterpret_cast<const float4*>(t_sm + (long)(hk0 * group / 2 + pair) * a.cq * ckp);
                    for (int tap = 0; tap < a.cq; ++tap, srow += ring.row) {
                        const float4 *e4 = reinterpret_cast<const float4*>(srow), *o4 = reinterpret_cast<const float4*>(srow + ring.half);
                        int at = q1;
                        float4 e = e4[at], o = o4[at];
                        for (int j = 0; j < ckp / 4; ++j, w += 2) {
                            at = at + 1 == ring.keys / 4 ? 0 : at + 1;
                            const float4 e1 = e4[at], o1 = o4[at], wa = w[0], wb = w[1];
                            const float2 s[7] = {make_float2(e.x, e.y), make_float2(e.z, e.w), make_float2(o.x, o.y), make_float2(o.z, o.w),
                                                 make_float2(e1.x, e1.y), make_float2(e1.z, e1.w), make_float2(o1.x, o1.y)};
                            const float2 ws[4] = {make_float2(wa.x, wa.y), make_float2(wa.z, wa.w), make_float2(wb.x, wb.y), make_float2(wb.z, wb.w)};
#pragma unroll
                            for (int t = 0; t < 4; ++t)
#pragma unroll
                                for (int k = 0; k < 4; ++k) z[k] = __ffma2_rn(ws[t], s[k + t], z[k]);
                            e = e1; o = o1;
                        }
                    }
                    float* to = c_sm + (((long)r * H + hk0 * group + 2 * pair) << a.shift) + 4 * quad;
                    *reinterpret_cast<float4*>(to) = make_float4(z[0].x, z[1].x, z[2].x, z[3].x);
                    if (2 * pair + 1 < heads) *reinterpret_cast<float4*>(to + tile) = make_float4(z[0].y, z[1].y, z[2].y, z[3].y);
                }
                __syncthreads();
            }
            // head mix and softmax statistics: (row, four heads, four keys) a thread; the threads of a row and four heads are neighbours
            for (int i0 = warp * 32; i0 < a.cq2 * oquads << (a.shift - 2); i0 += THREADS) {
                const int i = i0 + lane, kq = (i & (quads - 1)) * 4, rest = i >> (a.shift - 2), r0 = rest / oquads, o0 = (rest - r0 * oquads) * 4;
                const bool on = r0 < a.cq2;
                const int r = on ? r0 : 0;
                float z[4][4];
                mix_heads(z, W_sm + o0, c_sm + (((long)r * H) << a.shift) + kq, H, tile);
                const int seen = len - a.cq2 + r - k0 - kq;                          // of the four keys those up to this one are seen by the row
#pragma unroll
                for (int o = 0; o < 4; ++o) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k > seen) z[o][k] = -INFINITY;
                    const int row = r * H + o0 + o;
                    const bool put = on && o0 + o < H;
                    const float2 old = put ? ml[row] : make_float2(0.0f, 0.0f);
                    float top = fmaxf(fmaxf(z[o][0], z[o][1]), fmaxf(z[o][2], z[o][3]));
                    for (int s = 1; s < quads; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                    top = fmaxf(top, old.x);
                    // while a row has seen nothing its maximum is -inf and its sum 0
                    const float ref = top == -INFINITY ? 0.0f : top;
                    float sum = 0.0f;
#pragma unroll
                    for (int k = 0; k < 4; ++k) sum += fast_exp2(z[o][k] - ref);
                    for (int s = 1; s < quads; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
                    if (put) {
                        *reinterpret_cast<float4*>(a.logits + ((long)b * a.cq2 * H + row) * a.pitch + k0 + kq) = make_float4(z[o][0], z[o][1], z[o][2], z[o][3]);
                        if (kq == 0) ml[row] = make_float2(top, fmaf(old.y, fast_exp2(old.x - ref), sum));
                    }
                }
            }
            // the next tile's scores go to places of the ring that this tile's conv, two barriers back, was the last to read
        }
        __syncthreads();
        const long part = me + b;
        for (int i = threadIdx.x; i < a.cq2 * H; i += THREADS) a.part_ml[part * a.cq2 * H + i] = ml[i];
        __syncthreads();
        x = (long)before[b] + tb;
    }
}

// Tasks of (GT query heads, share of a tile's keys) are dealt to warps; where there are fewer heads than warps, `copies` warps share
// one and each keeps an output of its own.
template <typename T, int DMAX, int GT>
__global__ void __launch_bounds__(THREADS, sizeof(T) * DMAX > 256 ? 1 : 2) mta_decode_values_kernel(PagedCache c, MtaArgs a, int copies) {
    constexpr bool HALF = sizeof(T) == 2;
    using V = std::conditional_t<HALF, ValueTile<T, DMAX>, ValueTileF32<DMAX>>;
    using P = Pieces<GT>;
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int H = c.H, group = H / c.kv_heads, tile = 1 << a.shift, ckp = round4(a.ck2), left = (a.ck2 - 1) / 2, pp = prob_pitch(tile, a.ck2);
    const int quads = tile / 4, oquads = round4(H) / 4, ap = piece_pitch(tile);
    const ValueSmem m = value_smem(a.B, H, c.D, tile, a.cq2, a.ck2, copies);
    float *p_sm = reinterpret_cast<float*>(smem + m.p), *y_sm = reinterpret_cast<float*>(smem + m.y), *by = reinterpret_cast<float*>(smem + m.by);
    float *W_sm = reinterpret_cast<float*>(smem + m.W), *t_sm = reinterpret_cast<float*>(smem + m.taps), *o_sm = reinterpret_cast<float*>(smem + m.o);
    T* a_sm = reinterpret_cast<T*>(smem + m.a);                  // [head][piece][key], float32: [head][key]
    float2* ml = reinterpret_cast<float2*>(smem + m.ml);
    int *before = reinterpret_cast<int*>(smem + m.before), *lens = before + a.B + 1;

    // nothing up to pdl_wait() is written by the kernel before
    count_tiles(c, a.B, a.shift, before, lens);
    load_mix(W_sm, a.W2, H, a.w_dtype);
    for (int i = threadIdx.x; i < H * a.cq2 * ckp; i += THREADS) {
        const int j = i % ckp, row = i / ckp;
        t_sm[i] = j < a.ck2 ? load_weight(a.w2, (long)row * a.ck2 + j, a.w_dtype) : 0.0f;
    }
    __syncthreads();
    const T* pool = static_cast<const T*>(c.v);
    const long n = before[a.B], workers = n < a.workers ? n : a.workers, me = blockIdx.x;
    const long begin = run_begin(me, n, workers > 0 ? workers : 1), end = run_begin(me + 1, n, workers > 0 ? workers : 1);
    if (me < workers) {
        const int b = find_line(before, a.B, begin);
        prefetch_tile(c, pool, c.slot(b), (int)(begin - before[b]) << a.shift, tile, lens[b]);
    }
    if constexpr (std::is_same_v<T, __half>) {
        // Probabilities are at most 1, so a weight of head o is at most A = sum_h |W2[o,h]| sum |w2[h]|.  Times 2^14 over the power of two
        // below A it stays under 2^15, and its pieces are out of fp16's subnormal numbers down to 2^-28 A.
        for (int h = threadIdx.x; h < H; h += THREADS) {
            float s = 0.0f;
            for (int i = 0; i < a.cq2 * ckp; ++i) s += fabsf(t_sm[h * a.cq2 * ckp + i]);
            y_sm[h] = s;
        }
        __syncthreads();
        for (int o = threadIdx.x; o < H; o += THREADS) {
            float s = 0.0f;
            for (int h = 0; h < H; ++h) s = fmaf(fabsf(W_sm[h * round4(H) + o]), y_sm[h], s);
            by[o] = s > 1e-30f && s < 1e30f ? exp2f((float)(14 - ilogbf(s))) : 1.0f;
        }
        __syncthreads();
    }
    pdl_wait();
    if (me >= workers) return;

    for (long x = begin; x < end;) {
        const int b = find_line(before, a.B, x), len = lens[b], slot = c.slot(b), tiles = before[b + 1] - before[b];
        const int ta = (int)(x - before[b]), tb = (int)(end - before[b] < tiles ? end - before[b] : tiles);
        const long w0 = run_owner(before[b], n, workers), w1 = run_owner((long)before[b] + tiles - 1, n, workers);
        // maximum and one over the sum of every (row, head), from all runs of the sequence: eight lanes each
        for (int i0 = threadIdx.x / 8; i0 < (a.cq2 * H + 31) / 32 * 32; i0 += THREADS / 8) {
            const int i = i0 < a.cq2 * H ? i0 : a.cq2 * H - 1;
            float top = -INFINITY, sum = 0.0f;
            for (long w = w0 + threadIdx.x % 8; w <= w1; w += 8) {
                const float2 v = a.part_ml[(w + b) * a.cq2 * H + i];
                const float t = fmaxf(top, v.x), ref = t == -INFINITY ? 0.0f : t;
                sum = fmaf(sum, fast_exp2(top - ref), v.y * fast_exp2(v.x - ref));
                top = t;
            }
#pragma unroll
            for (int s = 1; s < 8; s <<= 1) {
                const float v = __shfl_xor_sync(0xffffffffu, top, s), l = __shfl_xor_sync(0xffffffffu, sum, s);
                const float t = fmaxf(top, v), ref = t == -INFINITY ? 0.0f : t;
                sum = sum * fast_exp2(top - ref) + l * fast_exp2(v - ref);
                top = t;
            }
            // a row before the first token has no keys: its probabilities are zero
            if (threadIdx.x % 8 == 0 && i0 < a.cq2 * H) ml[i] = len - a.cq2 + i / H < 0 ? make_float2(0.0f, 0.0f) : make_float2(top, 1.0f / sum);
        }
        for (int i = threadIdx.x; i < copies * H * c.D; i += THREADS) o_sm[i] = 0.0f;
        __syncthreads();
        for (int tl = ta; tl < tb; ++tl) {
            const int k0 = tl << a.shift;
            if (tl + 1 < tb) prefetch_tile(c, pool, slot, k0 + tile, tile, len);
            for (int row = warp; row < a.cq2 * H; row += WARPS) {
                const float2 s = ml[row];
                const float* from = a.logits + ((long)b * a.cq2 * H + row) * a.pitch;
                for (int col = lane; col < pp; col += 32) {
                    const int key = k0 - left + col;
                    p_sm[row * pp + col] = key >= 0 && key < len && col < tile + a.ck2 - 1 ? fast_exp2(from[key] - s.x) * s.y : 0.0f;
                }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < H << (a.shift - 2); i += THREADS) {
                const int quad = i & (quads - 1), h = i >> (a.shift - 2);
                float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int tap = 0; tap < a.cq2; ++tap) conv_row(z, p_sm + (tap * H + h) * pp + 4 * quad, t_sm + (h * a.cq2 + tap) * ckp, ckp);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k0 + 4 * quad + e >= len) z[e] = 0.0f;
                *reinterpret_cast<float4*>(y_sm + (h << a.shift) + 4 * quad) = make_float4(z[0], z[1], z[2], z[3]);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < oquads << (a.shift - 2); i += THREADS) {
                const int kq = (i & (quads - 1)) * 4, o0 = (i >> (a.shift - 2)) * 4;
                float z[4][4];
                mix_heads(z, W_sm + o0, y_sm + kq, H, tile);
#pragma unroll
                for (int o = 0; o < 4; ++o) {
                    if (o0 + o >= H) break;
                    if constexpr (HALF) {
                        float f[4][P::PIECES];
#pragma unroll
                        for (int k = 0; k < 4; ++k) split_pieces<T>(std::is_same_v<T, __half> ? z[o][k] * by[o0 + o] : z[o][k], f[k]);
#pragma unroll
                        for (int piece = 0; piece < P::PIECES; ++piece)
                            *reinterpret_cast<uint2*>(a_sm + ((o0 + o) * P::PIECES + piece) * ap + kq) =
                                make_uint2(pack2<T>(f[0][piece], f[1][piece]), pack2<T>(f[2][piece], f[3][piece]));
                    } else {
                        *reinterpret_cast<float4*>(a_sm + ((o0 + o) << a.shift) + kq) = make_float4(z[o][0], z[o][1], z[o][2], z[o][3]);
                    }
                }
            }
            __syncthreads();
            // product with the values
            const int units = tile / KEYS, tasks = H / GT * copies;
            for (int task = warp; task < tasks; task += WARPS) {
                const int copy = task % copies, h0 = task / copies * GT, hk = h0 / group;
                int u = copy * units / copies;
                const int live_units = (len - k0 + KEYS - 1) / KEYS, ub = (copy + 1) * units / copies < live_units ? (copy + 1) * units / copies : live_units;
                if (u >= ub) continue;
                V values;
                auto fetch = [&](int unit) {
                    const int key = k0 + unit * KEYS;
                    values.load(pool, c.at(slot, hk, key), len - key < KEYS ? len - key : KEYS, c.D, lane);
                };
                fetch(u);
                if constexpr (HALF) {
                    float acc[V::CHUNKS][4][4];
#pragma unroll
                    for (int i = 0; i < V::CHUNKS; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.0f;
                    const int y = g / P::STRIDE, piece = g % P::STRIDE;
                    const bool on = y < GT && piece < P::PIECES;
                    const uint32_t* col = reinterpret_cast<const uint32_t*>(a_sm + (on ? ((h0 + y) * P::PIECES + piece) * ap : 0)) + t4;
                    for (; u < ub; ++u) {
                        values.multiply(acc, on ? col[u * 8] : 0u, on ? col[u * 8 + 4] : 0u);
                        if (u + 1 < ub) fetch(u + 1);
                    }
                    // sum over the pieces; a head's columns are those of one lane (four heads) or of two, which then halve the elements
                    constexpr int CH = V::CHUNKS;
                    float f[CH][8];
#pragma unroll
                    for (int i = 0; i < CH; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j) { f[i][j] = acc[i][j][0] + acc[i][j][1]; f[i][j + 4] = acc[i][j][2] + acc[i][j][3]; }
                    const int head = h0 + t4 * 2 / P::STRIDE;
                    const bool mine = t4 * 2 / P::STRIDE < GT;
                    float* to = o_sm + ((long)copy * H + (mine ? head : 0)) * c.D;
                    const float back = std::is_same_v<T, __half> && mine ? 1.0f / by[head] : 1.0f;
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        const int e0 = i * 64 + g * 8;
                        if constexpr (P::STRIDE == 4) {
                            float h[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float give = t4 & 1 ? f[i][e] : f[i][e + 4], keep = t4 & 1 ? f[i][e + 4] : f[i][e];
                                h[e] = keep + __shfl_xor_sync(0xffffffffu, give, 1);
                            }
                            if (mine && e0 < c.D) {
                                float4* at = reinterpret_cast<float4*>(to + e0 + (t4 & 1) * 4);
                                float4 v = *at;
                                v.x = fmaf(h[0], back, v.x); v.y = fmaf(h[1], back, v.y); v.z = fmaf(h[2], back, v.z); v.w = fmaf(h[3], back, v.w);
                                *at = v;
                            }
                        } else if (e0 < c.D) {
#pragma unroll
                            for (int e = 0; e < 8; e += 4) {
                                float4* at = reinterpret_cast<float4*>(to + e0 + e);
                                float4 v = *at;
                                v.x = fmaf(f[i][e], back, v.x); v.y = fmaf(f[i][e + 1], back, v.y); v.z = fmaf(f[i][e + 2], back, v.z); v.w = fmaf(f[i][e + 3], back, v.w);
                                *at = v;
                            }
                        }
                    }
                } else {
                    float o[GT][4];
#pragma unroll
                    for (int y = 0; y < GT; ++y) o[y][0] = o[y][1] = o[y][2] = o[y][3] = 0.0f;
                    for (; u < ub; ++u) {
#pragma unroll
                        for (int i = 0; i < V::STEPS; ++i) {
                            float f[4];
                            unpack16<float>(values.r[i], f);
#pragma unroll
                            for (int y = 0; y < GT; ++y) {
                                const float p = a_sm[((h0 + y) << a.shift) + u * KEYS + i * V::SUBS + lane / V::ROWLANES];
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[y][e] = fmaf(p, f[e], o[y][e]);
                            }
                        }
                        if (u + 1 < ub) fetch(u + 1);
                    }
                    const int e0 = (lane % V::ROWLANES) * 4;
#pragma unroll
                    for (int y = 0; y < GT; ++y) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int s = V::ROWLANES; s < 32; s <<= 1) o[y][e] += __shfl_xor_sync(0xffffffffu, o[y][e], s);
                        if (lane < V::ROWLANES && e0 < c.D) {
                            float4* at = reinterpret_cast<float4*>(o_sm + ((long)copy * H + h0 + y) * c.D + e0);
                            float4 v = *at;
                            v.x += o[y][0]; v.y += o[y][1]; v.z += o[y][2]; v.w += o[y][3];
                            *at = v;
                        }
                    }
                }
            }
            // the next writes of p come after every thread's conv, those of y and of the weights behind the next barriers
        }
        __syncthreads();
        for (int i = threadIdx.x; i < H * c.D; i += THREADS) {
            float v = 0.0f;
            for (int y = 0; y < copies; ++y) v += o_sm[(long)y * H * c.D + i];
            if (w0 == w1) static_cast<T*>(a.out)[(long)b * H * c.D + i] = from_f32<T>(v);      // the only run of the sequence
            else a.part_o[(me + b) * H * c.D + i] = v;
        }
        __syncthreads();
        x = (long)before[b] + tb;
    }
}

// One block per (head, sequence): adds the runs' outputs in the order of their keys.  Sequences of no tokens get zeros.
template <typename T> __global__ void __launch_bounds__(128) mta_decode_join_kernel(PagedCache c, MtaArgs a) {
    extern __shared__ __align__(16) char smem[];
    int *before = reinterpret_cast<int*>(smem), *lens = before + a.B + 1;
    __shared__ float sum_o[4][256];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.x, b = blockIdx.y;
    count_tiles(c, a.B, a.shift, before, lens);
    __syncthreads();
    pdl_wait();
    T* out = static_cast<T*>(a.out) + ((long)b * c.H + h) * c.D;
    const int tiles = before[b + 1] - before[b];
    if (tiles == 0) {
        for (int d = threadIdx.x; d < c.D; d += 128) out[d] = from_f32<T>(0.0f);
        return;
    }
    const long n = before[a.B], workers = n < a.workers ? n : a.workers;
    const long w0 = run_owner(before[b], n, workers), w1 = run_owner((long)before[b] + tiles - 1, n, workers);
    if (w0 == w1) return;
    float4 o[2] = {make_float4(0, 0, 0, 0), make_float4(0, 0, 0, 0)};
#pragma unroll 4
    for (long w = w0 + warp; w <= w1; w += 4) {
        const float4* from = reinterpret_cast<const float4*>(a.part_o + ((w + b) * c.H + h) * c.D);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if ((lane + 32 * i) * 4 < c.D) {
                const float4 v = from[lane + 32 * i];
                o[i].x += v.x; o[i].y += v.y; o[i].z += v.z; o[i].w += v.w;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if ((lane + 32 * i) * 4 < c.D) *reinterpret_cast<float4*>(&sum_o[warp][(lane + 32 * i) * 4]) = o[i];
    __syncthreads();
    for (int d = threadIdx.x; d < c.D; d += 128) out[d] = from_f32<T>(sum_o[0][d] + sum_o[1][d] + sum_o[2][d] + sum_o[3][d]);
}

constexpr size_t SMEM_MOST = 227 * 1024;

struct Plan {
    int shift, kv_together, gt, copies, workers;
    size_t score_bytes, value_bytes;               // shared memory
    size_t ml_at, o_at, bytes;                     // workspace
    long pitch;
};

int make_plan(Plan* p, int B, int H, int kv_heads, int D, int cq, int ck, int cq2, int ck2, int max_length) {
    const int group = H / kv_heads;
    p->gt = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
    p->copies = 1;
    while (H / p->gt * p->copies * 2 <= WARPS) p->copies *= 2;
    bool fits = false;
    for (p->shift = 6; p->shift >= 4 && !fits; --p->shift) {
        const int tile = 1 << p->shift;
        for (p->kv_together = kv_heads; p->kv_together >= 1 && !fits; p->kv_together = p->kv_together / 2) {
            p->score_bytes = score_smem(B, H, group, p->kv_together, tile, cq, ck, cq2).bytes;
            p->value_bytes = value_smem(B, H, D, tile, cq2, ck2, p->copies).bytes;
            // a smaller tile before the heads are taken in parts (of whole pairs)
            fits = p->score_bytes <= SMEM_MOST && p->value_bytes <= SMEM_MOST && (p->kv_together == kv_heads || (p->shift == 4 && p->kv_together * group % 2 == 0));
            if (fits) break;
        }
        if (fits) break;
    }
    MTA_REQUIRE(fits, "mta_decode: %d heads of %d elements with kernels %dx%d and %dx%d need %zu and %zu bytes of shared memory, more than %zu", H, D, cq, ck,
                cq2, ck2, score_smem(B, H, group, 1, 16, cq, ck, cq2).bytes, value_smem(B, H, D, 16, cq2, ck2, p->copies).bytes, SMEM_MOST);
    const long tiles = (long)B * ((max_length + (1 << p->shift) - 1) >> p->shift);
    const long most = (long)DECODE_SMS * 2;
    p->workers = (int)(tiles < most ? (tiles < 1 ? 1 : tiles) : most);
    p->pitch = (max_length + 63) / 64 * 64;
    const size_t parts = (size_t)p->workers + B;
    p->ml_at = ((size_t)B * cq2 * H * p->pitch * 4 + 255) / 256 * 256;
    p->o_at = p->ml_at + (parts * cq2 * H * 8 + 255) / 256 * 256;
    p->bytes = p->o_at + parts * H * D * 4;
    return MTA_OK;
}

template <typename T, int DMAX, int NT> int launch_scores(const PagedCache& c, const MtaArgs& a, const Plan& p, cudaStream_t st) {
    return launch_kernel<mta_decode_scores_kernel<T, DMAX, NT>>("mta_decode_scores_kernel", dim3(p.workers), THREADS, p.score_bytes, st, c, a);
}

template <typename T, int DMAX> int launch_dim(const PagedCache& c, const MtaArgs& a, const Plan& p, cudaStream_t st) {
    const int R = a.cq + a.cq2 - 1;
    if (int rc = R <= 8 ? launch_scores<T, DMAX, 1>(c, a, p, st) : R <= 16 ? launch_scores<T, DMAX, 2>(c, a, p, st) : launch_scores<T, DMAX, 4>(c, a, p, st)) return rc;
    int rc = 0;
    if (p.gt == 4) rc = launch_kernel<mta_decode_values_kernel<T, DMAX, 4>>("mta_decode_values_kernel", dim3(p.workers), THREADS, p.value_bytes, st, c, a, p.copies);
    else if (p.gt == 2) rc = launch_kernel<mta_decode_values_kernel<T, DMAX, 2>>("mta_decode_values_kernel", dim3(p.workers), THREADS, p.value_bytes, st, c, a, p.copies);
    else rc = launch_kernel<mta_decode_values_kernel<T, DMAX, 1>>("mta_decode_values_kernel", dim3(p.workers), THREADS, p.value_bytes, st, c, a, p.copies);
    if (rc) return rc;
    return launch_kernel<mta_decode_join_kernel<T>>("mta_decode_join_kernel", dim3(c.H, a.B), 128, (2 * a.B + 1) * sizeof(int), st, c, a);
}

template <typename T> int launch(const PagedCache& c, const MtaArgs& a, const Plan& p, cudaStream_t st) {
    if (c.D <= 64) return launch_dim<T, 64>(c, a, p, st);
    if constexpr (sizeof(T) == 4) return launch_dim<T, 128>(c, a, p, st);
    else return c.D <= 128 ? launch_dim<T, 128>(c, a, p, st) : launch_dim<T, 256>(c, a, p, st);
}

}  // namespace

int mta_decode_workspace(int B, int H, int kv_heads, int D, int cq, int ck, int cq2, int ck2, int max_length, size_t* bytes) {
    Plan p;
    if (int rc = make_plan(&p, B, H, kv_heads, D, cq, ck, cq2, ck2, max_length)) return rc;
    *bytes = p.bytes;
    return MTA_OK;
}

int mta_decode_launch(const PagedCache& cache, const void* w1, const void* W1, const void* w2, const void* W2, int w_dtype, void* out, void* workspace, int B,
                      int cq, int ck, int cq2, int ck2, int dtype, cudaStream_t st) {
    PagedCache c = cache;
    if (int rc = wait_flag_ptr(&c.err)) return rc;
    Plan p;
    if (int rc = make_plan(&p, B, c.H, c.kv_heads, c.D, cq, ck, cq2, ck2, c.max_length)) return rc;
    MtaArgs a;
    a.w1 = w1; a.W1 = W1; a.w2 = w2; a.W2 = W2; a.w_dtype = w_dtype; a.out = out;
    char* ws = static_cast<char*>(workspace);
    a.logits = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + p.ml_at);
    a.part_o = reinterpret_cast<float*>(ws + p.o_at);
    a.pitch = p.pitch; a.B = B; a.cq = cq; a.ck = ck; a.cq2 = cq2; a.ck2 = ck2;
    a.scale = LOG2E / sqrtf((float)c.D);
    a.workers = p.workers; a.shift = p.shift; a.kv_together = p.kv_together;
    if (dtype == MTA_F32) return launch<float>(c, a, p, st);
    return dtype == MTA_BF16 ? launch<__nv_bfloat16>(c, a, p, st) : launch<__half>(c, a, p, st);
}

}  // namespace mta
