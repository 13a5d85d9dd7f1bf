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
//   scores  block = a run of key tiles, all heads: scores, conv, head mix; logits to the workspace (float32, in units of ln 2),
//           maximum and sum of every (row, head) of the run
//   values  the same runs: joins the maxima and sums of all runs, probabilities, conv, head mix, product with the values
//   join    adds the runs' outputs
// Keys and values are read once; the logits add 4 cq2 bytes written and read, mostly in L2, to the 4 D of keys and values in 16 bits.
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
    float scale;
    int workers, shift;    // key tiles of 1 << shift
    int kv_together;       // kv heads whose scores fit in shared memory at once
};

__host__ __device__ inline int taps_pitch(int ck) { return (ck + 3) / 4 * 4; }
__host__ __device__ inline int halo(int x) { return (x + KEYS - 1) / KEYS * KEYS; }

// Columns of the score tile: whole tiles of 16 keys to the left and right of the run's own, up to 3 columns that put the first window
// on a 16-byte boundary, and what the last window reads past its taps.  12 more than a multiple of 16: accumulator rows then
// fall on different banks.
__host__ __device__ inline int score_pitch(int tile, int ck) { return halo((ck - 1) / 2) + tile + halo(ck - 1 - (ck - 1) / 2) + 12; }
__host__ __device__ inline int prob_pitch(int tile, int ck2) { return tile + taps_pitch(ck2) + 4; }
__host__ __device__ inline int heads4(int H) { return (H + 3) / 4 * 4; }

struct ScoreSmem {
    size_t s, c, l, W, taps, ml, before, bytes;
};
__host__ __device__ inline ScoreSmem score_smem(int B, int H, int group, int kv_together, int tile, int cq, int ck, int cq2) {
    ScoreSmem m;
    size_t at = 0;
    const int R = cq + cq2 - 1;
    m.s = at; at += (size_t)kv_together * group * R * score_pitch(tile, ck) * 4;
    m.c = at; at += (size_t)cq2 * H * tile * 4;
    m.l = at; at += (size_t)cq2 * H * tile * 4;
    m.W = at; at += (size_t)H * heads4(H) * 4;
    m.taps = at; at += (size_t)H * cq * taps_pitch(ck) * 4;
    m.ml = at; at += ((size_t)cq2 * H * 8 + 15) / 16 * 16;
    m.before = at; at += (size_t)(2 * B + 1) * 4;
    m.bytes = at;
    return m;
}
struct ValueSmem {
    size_t p, y, a, W, taps, ml, o, before, bytes;
};
__host__ __device__ inline ValueSmem value_smem(int B, int H, int D, int tile, int cq2, int ck2, int copies) {
    ValueSmem m;
    size_t at = 0;
    m.p = at; at += (size_t)cq2 * H * prob_pitch(tile, ck2) * 4;
    m.y = at; at += (size_t)H * tile * 4;
    m.a = at; at += (size_t)H * tile * 4;
    m.W = at; at += (size_t)H * heads4(H) * 4;
    m.taps = at; at += (size_t)H * cq2 * taps_pitch(ck2) * 4;
    m.ml = at; at += ((size_t)cq2 * H * 8 + 15) / 16 * 16;
    m.o = at; at += (size_t)copies * H * D * 4;
    m.before = at; at += (size_t)(2 * B + 1) * 4;
    m.bytes = at;
    return m;
}

// What a block's run begins with: W transposed to [h][o] so that four outputs are one 16-byte load, taps padded with zeros.
__device__ __forceinline__ void load_mix(float* W, const void* from, int H, int w_dtype) {
    const int Hp = heads4(H);
    for (int i = threadIdx.x; i < H * Hp; i += THREADS) {
        const int h = i / Hp, o = i % Hp;
        W[i] = o < H ? load_weight(from, (long)o * H + h, w_dtype) : 0.0f;
    }
}
__device__ __forceinline__ void load_taps(float* taps, const void* from, int rows, int ck, int w_dtype) {
    const int ckp = taps_pitch(ck);
    for (int i = threadIdx.x; i < rows * ckp; i += THREADS) taps[i] = i % ckp < ck ? load_weight(from, (long)(i / ckp) * ck + i % ckp, w_dtype) : 0.0f;
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

// to[o][k] = sum_h W[h][o] from[h][k] for `tile` keys; four outputs a thread.  put(o, k, value).
template <typename PUT> __device__ __forceinline__ void mix_heads(const float* W, const float* from, int H, int shift, int item, PUT put) {
    const int Hp = heads4(H), k = item & ((1 << shift) - 1), o = (item >> shift) * 4;
    float4 z = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int h = 0; h < H; ++h) {
        const float x = from[(h << shift) + k];
        const float4 w = *reinterpret_cast<const float4*>(W + h * Hp + o);
        z.x = fmaf(w.x, x, z.x); z.y = fmaf(w.y, x, z.y); z.z = fmaf(w.z, x, z.z); z.w = fmaf(w.w, x, z.w);
    }
    put(o, k, z.x);
    if (o + 1 < H) put(o + 1, k, z.y);
    if (o + 2 < H) put(o + 2, k, z.z);
    if (o + 3 < H) put(o + 3, k, z.w);
}

template <typename T, int DMAX, int NT>
__global__ void __launch_bounds__(THREADS, 2) mta_decode_scores_kernel(PagedCache c, MtaArgs a) {
    using K = KeyTile<T, DMAX>;
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int H = c.H, group = H / c.kv_heads, tile = 1 << a.shift, R = a.cq + a.cq2 - 1, ckp = taps_pitch(a.ck);
    const int left = (a.ck - 1) / 2, hl = halo(left), hr = halo(a.ck - 1 - left), off = left & 3, pitch = score_pitch(tile, a.ck);
    const ScoreSmem m = score_smem(a.B, H, group, a.kv_together, tile, a.cq, a.ck, a.cq2);
    float *s_sm = reinterpret_cast<float*>(smem + m.s), *c_sm = reinterpret_cast<float*>(smem + m.c), *l_sm = reinterpret_cast<float*>(smem + m.l);
    float *W_sm = reinterpret_cast<float*>(smem + m.W), *t_sm = reinterpret_cast<float*>(smem + m.taps);
    float2* ml = reinterpret_cast<float2*>(smem + m.ml);
    int *before = reinterpret_cast<int*>(smem + m.before), *lens = before + a.B + 1;

    pdl_wait();
    count_tiles(c, a.B, a.shift, before, lens);
    load_mix(W_sm, a.W1, H, a.w_dtype);
    load_taps(t_sm, a.w1, H * a.cq, a.ck, a.w_dtype);
    // columns past the last tile are read with taps of zero: they have to be finite
    for (int i = threadIdx.x; i < a.kv_together * group * R * pitch; i += THREADS) s_sm[i] = 0.0f;
    __syncthreads();
    const long n = before[a.B], workers = n < a.workers ? n : a.workers, me = blockIdx.x;
    if (me >= workers) return;
    const long end = run_begin(me + 1, n, workers);
    const T* pool = static_cast<const T*>(c.k);
    const bool whole = a.kv_together == c.kv_heads;      // all heads at once: the columns that tiles share are kept

    for (long x = run_begin(me, n, workers); x < end;) {
        const int b = find_line(before, a.B, x), len = lens[b], slot = c.slot(b);
        const int ta = (int)(x - before[b]), tb = (int)(end - before[b] < before[b + 1] - before[b] ? end - before[b] : before[b + 1] - before[b]);
        for (int i = threadIdx.x; i < a.cq2 * H; i += THREADS) ml[i] = make_float2(-INFINITY, 0.0f);
        for (int tl = ta; tl < tb; ++tl) {
            const int k0 = tl << a.shift;
            for (int hk0 = 0; hk0 < c.kv_heads; hk0 += a.kv_together) {
                const int nk = c.kv_heads - hk0 < a.kv_together ? c.kv_heads - hk0 : a.kv_together;
                // scores of the key tiles that are not there yet, one (kv head, 16 keys) a warp and step
                const int first = whole && tl > ta ? k0 + hr : k0 - hl, units = (k0 + tile + hr - first) / KEYS, tasks = nk * units;
                K keys;
                auto fetch = [&](int task) {
                    const int key = first + task % units * KEYS, hk = hk0 + task / units;
                    const long base = key >= 0 && key < len ? c.at(slot, hk, key) : -1L;
                    keys.load(pool, base, len - key < KEYS ? len - key : KEYS, c.D, lane);
                };
                int task = warp * tasks / WARPS;
                const int last = (warp + 1) * tasks / WARPS;
                if (task < last) fetch(task);
                for (; task < last; ++task) {
                    const int key = first + task % units * KEYS, hk = task / units;
                    for (int gq = 0; gq < group; ++gq) {
                        float acc[NT][4];
                        const T* q = static_cast<const T*>(c.q_hist) + ((long)slot * c.ring * H + (hk0 + hk) * group + gq) * c.D;
                        keys.template score<NT>(acc, lane, [&](int row, int ch) {
                            const int pos = len - R + row, e = (ch * 4 + t4) * K::EPL;
                            return row < R && pos >= 0 && e < c.D ? *reinterpret_cast<const uint4*>(q + (long)(pos % c.ring) * H * c.D + e) : make_uint4(0, 0, 0, 0);
                        });
                        float* s = s_sm + (long)(hk * group + gq) * R * pitch + (key - k0 + hl + off);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                const int row = 8 * nt + 2 * t4 + (y & 1), kk = g + 8 * (y >> 1);
                                if (row < R) s[row * pitch + kk] = key + kk <= len - R + row ? acc[nt][y] * a.scale : 0.0f;
                            }
                        }
                    }
                    if (task + 1 < last) fetch(task + 1);
                }
                __syncthreads();
                const int quads = tile / 4, heads = nk * group;
                for (int i = threadIdx.x; i < heads * a.cq2 * quads; i += THREADS) {
                    const int quad = i % quads, hr_ = i / quads, h = hr_ % heads, r = hr_ / heads;
                    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    const float* s = s_sm + (long)(h * R + r) * pitch + 4 * quad + hl + off - left;
                    const float* w = t_sm + (hk0 * group + h) * a.cq * ckp;
                    for (int tap = 0; tap < a.cq; ++tap) conv_row(z, s + tap * pitch, w + tap * ckp, ckp);
                    *reinterpret_cast<float4*>(c_sm + (((long)r * H + hk0 * group + h) << a.shift) + 4 * quad) = make_float4(z[0], z[1], z[2], z[3]);
                }
                __syncthreads();
            }
            if (whole && tl + 1 < tb) {
                // the columns that the next tile shares move to its place
                const int keep = hl + hr;
                for (int row = warp; row < H * R; row += WARPS) {
                    float* s = s_sm + (long)row * pitch + off;
                    const float v = lane < keep ? s[tile + lane] : 0.0f;
                    __syncwarp();
                    if (lane < keep) s[lane] = v;
                }
            }
            for (int i = threadIdx.x; i < a.cq2 * (heads4(H) / 4) << a.shift; i += THREADS) {
                const int per = (heads4(H) / 4) << a.shift, r = i / per;
                float* l = l_sm + (((long)r * H) << a.shift);
                const int seen = len - a.cq2 + r - k0;                  // keys up to this one of the tile are seen by the row
                mix_heads(W_sm, c_sm + (((long)r * H) << a.shift), H, a.shift, i % per,
                          [&](int o, int k, float v) { l[(o << a.shift) + k] = k <= seen ? v * LOG2E : -INFINITY; });
            }
            __syncthreads();
            for (int row = warp; row < a.cq2 * H; row += WARPS) {
                const float* l = l_sm + ((long)row << a.shift);
                float* to = a.logits + ((long)b * a.cq2 * H + row) * a.pitch + k0;
                float top = -INFINITY, sum = 0.0f, v[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int k = lane + 32 * i;
                    v[i] = k < tile ? l[k] : -INFINITY;
                    if (k < tile && k0 + k < len) to[k] = v[i];
                    top = fmaxf(top, v[i]);
                }
#pragma unroll
                for (int s = 1; s < 32; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                const float2 old = ml[row];
                top = fmaxf(top, old.x);
                // while a row has seen nothing its maximum is -inf and its sum 0
                const float ref = top == -INFINITY ? 0.0f : top;
                sum = exp2f(v[0] - ref) + exp2f(v[1] - ref);
#pragma unroll
                for (int s = 1; s < 32; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
                if (lane == 0) ml[row] = make_float2(top, old.y * exp2f(old.x - ref) + sum);
            }
            // the next writes of l, c and ml are two barriers away, those of s behind the barrier after the mix
        }
        __syncthreads();
        const long part = me + b;
        for (int i = threadIdx.x; i < a.cq2 * H; i += THREADS) a.part_ml[part * a.cq2 * H + i] = ml[i];
        __syncthreads();
        x = (long)before[b] + tb;
    }
}

// kv heads are dealt to warps; where there are fewer than warps, `copies` warps share one and each keeps an output of its own.
template <typename T, int DMAX, int GT>
__global__ void __launch_bounds__(THREADS, 2) mta_decode_values_kernel(PagedCache c, MtaArgs a, int copies) {
    using V = ValueTile<T, DMAX>;
    constexpr int EPL = V::EPL;
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int H = c.H, group = H / c.kv_heads, tile = 1 << a.shift, ckp = taps_pitch(a.ck2), left = (a.ck2 - 1) / 2, pp = prob_pitch(tile, a.ck2);
    const ValueSmem m = value_smem(a.B, H, c.D, tile, a.cq2, a.ck2, copies);
    float *p_sm = reinterpret_cast<float*>(smem + m.p), *y_sm = reinterpret_cast<float*>(smem + m.y), *a_sm = reinterpret_cast<float*>(smem + m.a);
    float *W_sm = reinterpret_cast<float*>(smem + m.W), *t_sm = reinterpret_cast<float*>(smem + m.taps), *o_sm = reinterpret_cast<float*>(smem + m.o);
    float2* ml = reinterpret_cast<float2*>(smem + m.ml);
    int *before = reinterpret_cast<int*>(smem + m.before), *lens = before + a.B + 1;

    // none of this is written by the kernel before
    count_tiles(c, a.B, a.shift, before, lens);
    load_mix(W_sm, a.W2, H, a.w_dtype);
    load_taps(t_sm, a.w2, H * a.cq2, a.ck2, a.w_dtype);
    __syncthreads();
    pdl_wait();
    const long n = before[a.B], workers = n < a.workers ? n : a.workers, me = blockIdx.x;
    if (me >= workers) return;
    const long end = run_begin(me + 1, n, workers);
    const T* pool = static_cast<const T*>(c.v);

    for (long x = run_begin(me, n, workers); x < end;) {
        const int b = find_line(before, a.B, x), len = lens[b], slot = c.slot(b), tiles = before[b + 1] - before[b];
        const int ta = (int)(x - before[b]), tb = (int)(end - before[b] < tiles ? end - before[b] : tiles);
        const long w0 = run_owner(before[b], n, workers), w1 = run_owner((long)before[b] + tiles - 1, n, workers);
        // maximum and one over the sum of every (row, head), from all runs of the sequence: eight lanes each
        for (int i0 = threadIdx.x / 8; i0 < (a.cq2 * H + 31) / 32 * 32; i0 += THREADS / 8) {
            const int i = i0 < a.cq2 * H ? i0 : a.cq2 * H - 1;
            float top = -INFINITY, sum = 0.0f;
            for (long w = w0 + threadIdx.x % 8; w <= w1; w += 8) top = fmaxf(top, a.part_ml[(w + b) * a.cq2 * H + i].x);
#pragma unroll
            for (int s = 1; s < 8; s <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
            for (long w = w0 + threadIdx.x % 8; w <= w1; w += 8) {
                const float2 v = a.part_ml[(w + b) * a.cq2 * H + i];
                sum += v.y * exp2f(v.x - top);
            }
#pragma unroll
            for (int s = 1; s < 8; s <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
            // a row before the first token has no keys: its probabilities are zero
            if (threadIdx.x % 8 == 0 && i0 < a.cq2 * H) ml[i] = len - a.cq2 + i / H < 0 ? make_float2(0.0f, 0.0f) : make_float2(top, 1.0f / sum);
        }
        for (int i = threadIdx.x; i < copies * H * c.D; i += THREADS) o_sm[i] = 0.0f;
        __syncthreads();
        for (int tl = ta; tl < tb; ++tl) {
            const int k0 = tl << a.shift;
            for (int i = threadIdx.x; i < a.cq2 * H * pp; i += THREADS) {
                const int col = i % pp, row = i / pp, key = k0 - left + col;
                float v = 0.0f;
                if (key >= 0 && key < len && col < tile + a.ck2 - 1 && len - a.cq2 + row / H >= 0) {
                    const float2 s = ml[row];
                    v = exp2f(a.logits[((long)b * a.cq2 * H + row) * a.pitch + key] - s.x) * s.y;
                }
                p_sm[i] = v;
            }
            __syncthreads();
            const int quads = tile / 4;
            for (int i = threadIdx.x; i < H * quads; i += THREADS) {
                const int quad = i % quads, h = i / quads;
                float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int tap = 0; tap < a.cq2; ++tap) conv_row(z, p_sm + (long)(tap * H + h) * pp + 4 * quad, t_sm + (h * a.cq2 + tap) * ckp, ckp);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k0 + 4 * quad + e >= len) z[e] = 0.0f;
                *reinterpret_cast<float4*>(y_sm + (h << a.shift) + 4 * quad) = make_float4(z[0], z[1], z[2], z[3]);
            }
            __syncthreads();
            for (int i = threadIdx.x; i < (heads4(H) / 4) << a.shift; i += THREADS)
                mix_heads(W_sm, y_sm, H, a.shift, i, [&](int o, int k, float v) { a_sm[(o << a.shift) + k] = v; });
            __syncthreads();
            // product with the values: (GT query heads, share of the tile's units) per task
            const int units = tile / KEYS, tasks = H / GT * copies;
            for (int task = warp; task < tasks; task += WARPS) {
                const int copy = task % copies, h0 = task / copies * GT, hk = h0 / group;
                const int ua = copy * units / copies, ub = (copy + 1) * units / copies;
                float o[GT][EPL];
#pragma unroll
                for (int y = 0; y < GT; ++y)
#pragma unroll
                    for (int e = 0; e < EPL; ++e) o[y][e] = 0.0f;
                for (int u = ua; u < ub; ++u) {
                    const int key = k0 + u * KEYS;
                    if (key >= len) break;
                    V values;
                    values.load(pool, c.at(slot, hk, key), len - key < KEYS ? len - key : KEYS, c.D, lane);
#pragma unroll
                    for (int i = 0; i < V::STEPS; ++i) {
                        float f[EPL];
                        unpack16<T>(values.r[i], f);
#pragma unroll
                        for (int y = 0; y < GT; ++y) {
                            const float p = a_sm[((h0 + y) << a.shift) + u * KEYS + i * V::SUBS + lane / V::ROWLANES];
#pragma unroll
                            for (int e = 0; e < EPL; ++e) o[y][e] = fmaf(p, f[e], o[y][e]);
                        }
                    }
                }
                const int e0 = (lane % V::ROWLANES) * EPL;
#pragma unroll
                for (int y = 0; y < GT; ++y) {
#pragma unroll
                    for (int e = 0; e < EPL; ++e)
#pragma unroll
                        for (int s = V::ROWLANES; s < 32; s <<= 1) o[y][e] += __shfl_xor_sync(0xffffffffu, o[y][e], s);
                    if (lane < V::ROWLANES && e0 < c.D) {
                        float4* to = reinterpret_cast<float4*>(o_sm + ((long)copy * H + h0 + y) * c.D + e0);
#pragma unroll
                        for (int e = 0; e < EPL; e += 4) {
                            float4 v = to[e / 4];
                            v.x += o[y][e]; v.y += o[y][e + 1]; v.z += o[y][e + 2]; v.w += o[y][e + 3];
                            to[e / 4] = v;
                        }
                    }
                }
            }
            // p is written again after this tile's last reader of it; y and a behind the next barriers
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
            // a smaller tile before the heads are taken in parts, except at the smallest
            fits = p->score_bytes <= SMEM_MOST && p->value_bytes <= SMEM_MOST && (p->kv_together == kv_heads || p->shift == 4);
            if (fits) break;
        }
        if (fits) break;
    }
    MTA_REQUIRE(fits, "mta_decode: %d heads of %d elements with kernels %dx%d and %dx%d need %zu and %zu bytes of shared memory, more than %zu", H, D, cq, ck,
                cq2, ck2, score_smem(B, H, group, 1, 16, cq, ck, cq2).bytes, value_smem(B, H, D, 16, cq2, ck2, p->copies).bytes, SMEM_MOST);
    const long tiles = (long)B * ((max_length + (1 << p->shift) - 1) >> p->shift);
    const long most = (long)DECODE_SMS * 3;
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
    a.scale = 1.0f / sqrtf((float)c.D);
    a.workers = p.workers; a.shift = p.shift; a.kv_together = p.kv_together;
    if (dtype == MTA_F32) return launch<float>(c, a, p, st);
    return dtype == MTA_BF16 ? launch<__nv_bfloat16>(c, a, p, st) : launch<__half>(c, a, p, st);
}

}  // namespace mta
