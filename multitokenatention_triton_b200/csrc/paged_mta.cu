// The MTA module for one new token per sequence over a paged cache.  With t the newest token, R = cq + cq2 - 1 and pos(j) = t-R+1+j:
//
//   s[h,j,k] = scale * q[h,pos(j)] . k[h,k] for 0 <= k <= pos(j), else 0           j < R
//   c[h,r,k] = sum_{i,j} w1[h,i,j] s[h,r+i,k+j-(ck-1)/2]                           r < cq2
//   l[o,r,k] = sum_h W1[o,h] c[h,r,k];  p[o,r,.] = softmax over k <= pos(cq-1+r); a row before the first token has p = 0
//   y[h,k]   = sum_{i,j} w2[h,i,j] p[h,i,k+j-(ck2-1)/2],  k <= t
//   out[o]   = sum_k (sum_h W2[o,h] y[h,k]) v[o,k]
//
// The rows before the newest are computed again from the last R queries instead of being kept: an mma has sixteen query rows
// anyway, so they cost no byte more, and a cache that holds keys, values and R queries can be forked or moved at any token.
// Both head mixes need all heads of a key, the softmax all keys of a row, so the work is three kernels:
//   scores  block = a run of key tiles, all heads: scores, conv, head mix; logits to the workspace (float32, base 2),
//           maximum and sum of every (row, head) of the run
//   values  the same runs: joins the maxima and sums of all runs, probabilities, conv, head mix, product with the values
//   join    adds the runs' outputs
// Keys and values are read once; the logits add 4 cq2 bytes written and read, mostly in L2, to the 4 D of keys and values in 16 bits.
//
// Measured, bf16, D 128, taps 6x11 and 3x3 (a graph of calls): 16 sequences of 8192 tokens, 32 heads 475 us, 4.52 TB/s of keys and values
// (scores 274, values 220, join 7 under the profiler); 8 sequences of 1024 to 4096 tokens, 16 heads 83 us; one of 301 tokens 27 us.
// The long batch is bound by instructions and their latency (scores, when they took 291 us: 276 with every load from L1, 213 with no convs
// and mixes), the short ones by the chain of stages: a run of 155 keys has three.
#include <type_traits>

#include "paged.cuh"

namespace mta {
namespace {

// A block is one per SM, half of its warps on memory and half on arithmetic: eight stream keys (values) and multiply, eight run the
// convs, head mixes and softmaxes of the tile before (after).  Two blocks of eight warps that did one after the other left the
// memory idle in every block's second half: 770 us for the long batch.  Asking L2 for the next tile ahead made it slower (1.47 GB
// read from memory instead of 1.11).
constexpr int ROLE_WARPS = 8, ROLE_THREADS = ROLE_WARPS * 32, THREADS = 2 * ROLE_THREADS;
// Named barriers: a stage's buffer is full or empty (by the stage's parity), and those of one half alone.
enum { BAR_FULL = 1, BAR_EMPTY = 3, BAR_MATH = 5, BAR_MEMORY = 6 };

struct MtaArgs {
    const void *w1, *W1, *w2, *W2;
    void* out;
    float* logits;         // (B, cq2, H, pitch)
    float2* part_ml;       // (parts, cq2, H)
    float* part_o;         // (parts, H, D)
    long pitch;
    int w_dtype, B, cq, ck, cq2, ck2;
    float scale;           // log2(e) / sqrt(D), taken into the first conv's taps: logits are in base 2
    int workers, shift;    // tiles of 1 << shift keys; runs are cut between any 16
    // The scores kernel's heads of keys: kv heads, or each of them `split` times, with a share of its query heads each, where one's query heads
    // are too many; and how many of them have scores that fit in shared memory at once.
    int score_heads, per_split, kv_together;       // head h of keys is kv head h * per_split >> 16
};

__host__ __device__ inline int round4(int x) { return (x + 3) / 4 * 4; }
__host__ __device__ inline int halo(int x) { return (x + KEYS - 1) / KEYS * KEYS; }

// The scores of two tiles and their neighbours: a ring of `keys` positions, so that one tile's scores are written while the conv reads
// the other's, and what tiles share is computed once; keys lie at their number plus a multiple of 16 that lets a sequence begin
// where the one before ended.  Where not all heads fit, the tiles (of one group of heads after another) have a ring each.  Two heads
// stand side by side, which lets one packed FMA serve both.  Keys (4i, 4i + 1) lie in the first half of a row, (4i + 2, 4i + 3) in
// the second, 16 bytes each: the conv's threads, four keys apart, read neighbouring 16 bytes.  The pads put the rows and halves
// that an accumulator writes at once into different banks.
// Windows begin on multiples of four keys: taps have up to three zeros in front (`lead`) for that, and zeros behind up to `taps`.
__host__ __device__ inline int lead(int ck) { return (4 - (ck - 1) / 2 % 4) % 4; }
__host__ __device__ inline int score_taps(int ck) { return round4(ck + lead(ck)); }
// Keys behind a tile that its windows touch, those that meet zeros included: they have to be scores of the same sequence, since a zero times
// what another sequence left there is no zero where that is not finite.
__host__ __device__ inline int halo_right(int ck) { return halo(score_taps(ck) - (ck - 1) / 2 - lead(ck)); }
// From one pair of heads' taps to the next pair's: 16 bytes more than they take, so that pairs lie in different banks.
__host__ __device__ inline int pair_taps(int cq, int ck) { return cq * score_taps(ck) + 2; }
struct ScoreRing {
    int keys, half, row;   // floats of half a row and of a row
    __host__ __device__ ScoreRing(int tile, int ck, bool whole) {
        keys = (halo((ck - 1) / 2) + tile + halo_right(ck)) * (whole ? 2 : 1);
        half = keys + (keys % 32 == 0 ? 8 : 24);
        row = 2 * half + 8;
    }
};
__host__ __device__ inline int prob_pitch(int tile, int ck2) { return tile + round4(ck2) + 4; }

struct ScoreSmem {
    size_t s, s_one, c, W, taps, ml, q_at, before, bytes;
};
__host__ __device__ inline ScoreSmem score_smem(int B, int H, int group, int kv_heads, int kv_together, int tile, int cq, int ck, int cq2) {
    ScoreSmem m;
    size_t at = 0;
    const int R = cq + cq2 - 1;
    const bool whole = kv_together == kv_heads;
    m.s_one = (size_t)((kv_together * group + 1) / 2) * R * ScoreRing(tile, ck, whole).row * 4;
    m.s = at; at += m.s_one * (whole ? 1 : 2);
    m.c = at; at += (size_t)cq2 * H * tile * 4;
    m.W = at; at += (size_t)H * round4(H) * 4;
    m.taps = at; at += (size_t)((H + 1) / 2) * pair_taps(cq, ck) * 8;
    m.ml = at; at += (size_t)cq2 * H * (tile / 4) * 8;
    m.q_at = at; at += (size_t)ROLE_WARPS * DECODE_MAX_ROWS * 8;
    m.before = at; at += (size_t)(2 * B + 1) * 4;
    m.bytes = at;
    return m;
}
// 16-bit pieces of the weights in a row of `tile` keys; the pad spreads eight rows over the banks.
__host__ __device__ inline int piece_pitch(int tile) { return tile + 8; }
struct ValueSmem {
    size_t p, y, a, a_one, W, taps, run_taps, ml, by, o, before, bytes;
};
__host__ __device__ inline ValueSmem value_smem(int B, int H, int D, int tile, int cq2, int ck2, int copies) {
    ValueSmem m;
    size_t at = 0;
    m.p = at; at += (size_t)cq2 * H * prob_pitch(tile, ck2) * 4;
    m.y = at; at += (size_t)H * tile * 4;
    m.a_one = (size_t)H * (3 * piece_pitch(tile) * 2);           // three pieces; float32: 4 bytes a key
    m.a = at; at += 2 * m.a_one;
    m.W = at; at += (size_t)H * round4(H) * 4;
    m.taps = at; at += (size_t)H * cq2 * round4(ck2) * 4;
    m.run_taps = at; at += (size_t)H * cq2 * round4(ck2) * 4;
    m.ml = at; at += ((size_t)cq2 * H * 4 + 15) / 16 * 16;
    m.by = at; at += (size_t)round4(H) * 4;
    m.o = at; at += (size_t)copies * H * D * 4;
    m.before = at; at += (size_t)(2 * B + 1) * 4;
    m.bytes = at;
    return m;
}

// W transposed to [h][o], so that four outputs are one 16-byte load.
__device__ __forceinline__ void load_mix(float* W, const void* from, int H, int w_dtype) {
    const int Hp = round4(H);
    for (int i = threadIdx.x % ROLE_THREADS; i < H * Hp; i += ROLE_THREADS) {
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

// The first conv of a stage: (two heads, row, four keys) a thread, sixteen packed FMAs for every four taps.  CHUNKS: quads of taps, 0 when
// there are more than the kernel has registers for; otherwise a tap row's whole window is loaded before its first FMA, so
// that the loads' latency is waited for once a row.
template <int CHUNKS> __device__ __forceinline__ void conv_pairs(const float* s, const float2* taps, float* to, const ScoreRing& ring, int q0, int heads, int H, int R,
                                                                 int cq, int cq2, int ckp, int shift, int tid) {
    const int quads = 1 << (shift - 2), pairs = (heads + 1) / 2, wrap = ring.keys / 4;
    for (int i = tid; i < pairs * cq2 * quads; i += ROLE_THREADS) {
        const int quad = i & (quads - 1), rest = i >> (shift - 2), r = rest / pairs, pair = rest - r * pairs;
        int at[CHUNKS + 1];
        at[0] = q0 + quad;
        if (at[0] >= wrap) at[0] -= wrap;
#pragma unroll
        for (int j = 1; j <= CHUNKS; ++j) at[j] = at[j - 1] + 1 == wrap ? 0 : at[j - 1] + 1;
        float2 z[4];
        z[0] = z[1] = z[2] = z[3] = make_float2(0.0f, 0.0f);
        const float* row = s + (pair * R + r) * ring.row;
        const float4* w = reinterpret_cast<const float4*>(taps + pair * (cq * ckp + 2));
        auto step = [&](const float4& e, const float4& o, const float4& e1, const float4& o1, const float4& wa, const float4& wb) {
            const float2 v[7] = {make_float2(e.x, e.y), make_float2(e.z, e.w), make_float2(o.x, o.y), make_float2(o.z, o.w),
                                 make_float2(e1.x, e1.y), make_float2(e1.z, e1.w), make_float2(o1.x, o1.y)};
            const float2 ws[4] = {make_float2(wa.x, wa.y), make_float2(wa.z, wa.w), make_float2(wb.x, wb.y), make_float2(wb.z, wb.w)};
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) z[k] = __ffma2_rn(ws[t], v[k + t], z[k]);
        };
        for (int tap = 0; tap < cq; ++tap, row += ring.row) {
            const float4 *e4 = reinterpret_cast<const float4*>(row), *o4 = reinterpret_cast<const float4*>(row + ring.half);
            if constexpr (CHUNKS > 0) {
                float4 e[CHUNKS + 1], o[CHUNKS + 1];
#pragma unroll
                for (int j = 0; j <= CHUNKS; ++j) { e[j] = e4[at[j]]; o[j] = o4[at[j]]; }
#pragma unroll
                for (int j = 0; j < CHUNKS; ++j) step(e[j], o[j], e[j + 1], o[j + 1], w[2 * j], w[2 * j + 1]);
                w += 2 * CHUNKS;
            } else {
                int x = at[0];
                float4 e = e4[x], o = o4[x];
                for (int j = 0; j < ckp / 4; ++j, w += 2) {
                    x = x + 1 == wrap ? 0 : x + 1;
                    const float4 e1 = e4[x], o1 = o4[x];
                    step(e, o, e1, o1, w[0], w[1]);
                    e = e1; o = o1;
                }
            }
        }
        float* out = to + ((r * H + 2 * pair) << shift) + 4 * quad;
        *reinterpret_cast<float4*>(out) = make_float4(z[0].x, z[1].x, z[2].x, z[3].x);
        if (2 * pair + 1 < heads) *reinterpret_cast<float4*>(out + (1 << shift)) = make_float4(z[0].y, z[1].y, z[2].y, z[3].y);
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

// Keys [k0, k1) of a sequence, of one block's run.
struct Span {
    int b, len, slot, k0, k1;
};
// The span that begins with unit x (16 keys) of a run that ends with unit `end`.
__device__ __forceinline__ Span span_at(const PagedCache& c, const int* before, const int* lens, int B, long x, long end) {
    Span s;
    s.b = find_line(before, B, x);
    s.len = lens[s.b];
    s.slot = c.slot(s.b);
    s.k0 = (int)(x - before[s.b]) * KEYS;
    s.k1 = (int)(end < before[s.b + 1] ? end - before[s.b] : before[s.b + 1] - before[s.b]) * KEYS;
    return s;
}

// What is added to key numbers for their places in the ring: key `first` comes to place `to` (a multiple of 16 each), no place is negative.
__device__ __forceinline__ int ring_turn(const ScoreRing& ring, bool whole, int to, int first) {
    if (!whole) { to = 0; }
    int turn = (to - first) % ring.keys;
    if (turn < 0) turn += ring.keys;
    return first + turn < 0 ? turn + ring.keys : turn;
}

// Where the 16 keys of lane `unit` of a stage lie for kv head 0; pages are looked up one stage ahead of their use.
struct Pages {
    int page;
    __device__ void look_up(const PagedCache& c, int slot, int key, bool on) {
        page = on ? __ldg(c.table + (long)slot * c.table_width + (key >> c.page_shift)) : -1;
    }
    __device__ long at(const PagedCache& c, int key, bool on) const {
        if (!on) return -1;
        if ((unsigned)page >= (unsigned)c.pages) { c.bad(); return -1; }
        return ((((long)page * c.kv_heads) << c.page_shift) + (key & ((1 << c.page_shift) - 1))) * c.D;
    }
};

// Tiles of 16 keys or values that a warp's task has and its registers hold in flight: as many as fit.  One at a time left the memory at
// 3.4 TB/s, and what a task costs besides its loads and products is paid half as often.
template <typename T, int DMAX, int NT = 1> constexpr int TOGETHER = sizeof(T) * DMAX <= 256 && NT <= 2 ? 2 : 1;

// The registers of a block are dealt anew once the roles part: 168 to a thread of the memory half, 88 to one of the other, 128 * 512 in all.
// In 16 bits that holds a head's queries and keys (values) up to D 128 at any number of rows and D 256 up to 8.  What needs more spills: D 256
// with 16 rows 148 bytes of stores a thread, with 32 rows (128 registers of queries, 64 of keys) 1.7 KB, its values kernels 108; float32 64 to
// 396 in the scores kernel of heads up to 64, up to 108 above.
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 168;"); }
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 88;"); }

template <typename T, int DMAX, int NT>
__global__ void __launch_bounds__(THREADS, 1) mta_decode_scores_kernel(PagedCache c, MtaArgs a) {
    constexpr bool HALF = sizeof(T) == 2;
    using K = KeyTile<T, DMAX>;
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int H = c.H, group = H / a.score_heads, tile = 1 << a.shift, R = a.cq + a.cq2 - 1, ckp = score_taps(a.ck);
    const int left = (a.ck - 1) / 2, hl = halo(left), hr = halo_right(a.ck), first_tap = lead(a.ck);
    const bool whole = a.kv_together == a.score_heads;           // all heads at once: what tiles share stays in the ring
    const ScoreRing ring(tile, a.ck, whole);
    const ScoreSmem m = score_smem(a.B, H, group, a.score_heads, a.kv_together, tile, a.cq, a.ck, a.cq2);
    float *s_sm = reinterpret_cast<float*>(smem + m.s), *c_sm = reinterpret_cast<float*>(smem + m.c), *W_sm = reinterpret_cast<float*>(smem + m.W);
    const int s_other = whole ? 0 : (int)(m.s_one / 4);          // from one stage's ring to the next one's
    float2 *t_sm = reinterpret_cast<float2*>(smem + m.taps), *ml = reinterpret_cast<float2*>(smem + m.ml);
    int *before = reinterpret_cast<int*>(smem + m.before), *lens = before + a.B + 1;

    // places that hold no score yet are read for keys behind the run, whose results are dropped: zeros, so that nothing undefined is read
    for (int i = threadIdx.x; i < (int)((m.c - m.s) / 16); i += THREADS) reinterpret_cast<float4*>(s_sm)[i] = make_float4(0, 0, 0, 0);
    pdl_wait();
    count_tiles(c, a.B, 4, before, lens);
    __syncthreads();
    const long n = before[a.B], workers = n < a.workers ? n : a.workers, me = blockIdx.x;
    if (me >= workers) return;
    const long begin = run_begin(me, n, workers), end = run_begin(me + 1, n, workers);

    if (warp < ROLE_WARPS) {
        // ---- scores.  A stage is a tile and a group of heads; a task one kv head and 16 or 32 keys of it.
        more_registers();
        const T* pool = static_cast<const T*>(c.k);
        const T* queries = static_cast<const T*>(c.q_hist);
        const int head_stride = c.D << c.page_shift;
        constexpr int N = TOGETHER<T, DMAX, NT>;
        long* q_at = reinterpret_cast<long*>(smem + m.q_at) + warp * DECODE_MAX_ROWS;       // this warp's query rows
        // Where the loads are, one task ahead of the arithmetic.
        struct Cursor {
            Span s;
            long at;           // of this lane's unit
            int k0, hk0, first, units, hk, unit, tasks_left, stage, turn, place;
            Pages next;
            bool done;
        } cur = {};
        auto first_of = [&](int k0) { return k0 + (whole && k0 > cur.s.k0 ? hr : -hl); };
        auto units_of = [&](int k0) { return ((k0 + tile < cur.s.k1 ? k0 + tile : cur.s.k1) + hr - first_of(k0)) / KEYS; };
        auto enter_stage = [&] {
            cur.first = first_of(cur.k0);
            cur.units = units_of(cur.k0);
            cur.place = (cur.first + cur.turn) % ring.keys;
            const int nk = a.score_heads - cur.hk0 < a.kv_together ? a.score_heads - cur.hk0 : a.kv_together;
            const int per_head = (cur.units + N - 1) / N, tasks = nk * per_head, t0 = warp * tasks / ROLE_WARPS;
            cur.tasks_left = (warp + 1) * tasks / ROLE_WARPS - t0;
            cur.hk = t0 / per_head;
            cur.unit = (t0 - cur.hk * per_head) * N;
            const int key = cur.first + lane * KEYS;
            const bool on = lane < cur.units && key >= 0 && key < cur.s.len;
            if (!whole || cur.k0 == cur.s.k0) cur.next.look_up(c, cur.s.slot, key, on);
            cur.at = cur.next.at(c, key, on);
            if (whole) {                                         // the next tile of the span
                const int ahead = cur.k0 + tile + hr + lane * KEYS;
                cur.next.look_up(c, cur.s.slot, ahead, lane < tile / KEYS && ahead < cur.s.len);
            }
        };
        auto enter_span = [&](long x, int place) {
            cur.s = span_at(c, before, lens, a.B, x, end);
            cur.k0 = cur.s.k0;
            cur.hk0 = 0;
            cur.turn = ring_turn(ring, whole, place, cur.s.k0 - hl);
        };
        enter_span(begin, 0);
        enter_stage();
        K keys[N];
        int task_unit = 0, task_hk = 0;                          // whose keys are on their way or next
        long next_at[N];                                         // where those lie, -1: nowhere
        int next_live = 0;
        // Sets the next task; load(i) then starts the loads of its i-th 16 keys.
        auto advance = [&]() -> bool {
            while (!cur.done && cur.tasks_left == 0) {
                ++cur.stage;
                cur.hk0 += a.kv_together;
                if (cur.hk0 >= a.score_heads) {
                    cur.hk0 = 0;
                    cur.k0 += tile;
                    if (cur.k0 >= cur.s.k1) {
                        const long x = (long)before[cur.s.b] + cur.s.k1 / KEYS;
                        if (x >= end) { cur.done = true; break; }
                        enter_span(x, cur.k0 + hr + cur.turn);   // behind the places of the span's last tile
                    }
                }
                enter_stage();
            }
            if (cur.done) return false;
            task_unit = cur.unit;
            task_hk = cur.hk;
            const long head = (long)((cur.hk0 + cur.hk) * a.per_split >> 16) * head_stride;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const long base = __shfl_sync(0xffffffffu, cur.at, cur.unit + i);    // -1 behind the last unit
                next_at[i] = base < 0 ? base : base + head;
            }
            next_live = cur.s.len - (cur.first + cur.unit * KEYS);
            cur.unit += N;
            if (cur.unit >= cur.units) { cur.unit = 0; ++cur.hk; }
            --cur.tasks_left;
            return true;
        };
        auto load = [&](int i) { keys[i].load(pool, next_at[i], next_live - i * KEYS, c.D, lane); };
        int stage = 0, span_b = -1, q_head = -1;
        constexpr int PARTS = K::template PARTS<NT * 8>;
        uint4 q[HALF ? PARTS / 2 : 1][HALF ? 2 * K::CH : 1];     // the A operands of a head
        // The span's query rows, and the queries of one head as A operands.
        auto query_rows = [&] {
            if (cur.s.b == span_b) return;
            __syncwarp();
            const int pos = cur.s.len - R + lane;
            q_at[lane] = lane < R && pos >= 0 ? ((long)cur.s.slot * c.ring + pos % c.ring) * H * c.D : -1;
            span_b = cur.s.b;
            q_head = -1;
            __syncwarp();
        };
        auto need_queries = [&](int head) {
            if constexpr (HALF) {
                if (q_head == head) return;
                q_head = head;
                const T* qh = queries + (long)head * c.D;
#pragma unroll
                for (int m_ = 0; m_ < PARTS / 2; ++m_) {
                    const long r0 = q_at[16 * m_ + g], r1 = NT > 1 ? q_at[16 * m_ + 8 + g] : -1;
#pragma unroll
                    for (int ch = 0; ch < K::CH; ++ch) {
                        const int e = K::element(ch, t4);
                        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
                        if (r0 >= 0 && e < c.D) lo = __ldg(reinterpret_cast<const uint4*>(qh + r0 + e));
                        if (NT > 1 && r1 >= 0 && e < c.D) hi = __ldg(reinterpret_cast<const uint4*>(qh + r1 + e));
                        q[m_][2 * ch] = make_uint4(lo.x, hi.x, lo.y, hi.y);
                        q[m_][2 * ch + 1] = make_uint4(lo.z, hi.z, lo.w, hi.w);
                    }
                }
            }
        };
        bool more = advance();
        if (more) {
#pragma unroll
            for (int i = 0; i < N; ++i) load(i);
            query_rows();
            need_queries((cur.hk0 + task_hk) * group);
        }
        // Scores of one task into the ring; the registers of its keys and queries take the next task's as soon as they are free.
        while (more) {
            // the cursor still stands where this task's keys lie
            while (stage < cur.stage) {
                barrier_arrive(BAR_FULL + (stage & 1), THREADS);
                ++stage;
                if (stage >= 2) barrier_sync(BAR_EMPTY + (stage & 1), THREADS);
            }
            const int len = cur.s.len;
            const int first_key = cur.first + task_unit * KEYS, local = task_hk * group, head0 = (cur.hk0 + task_hk) * group;
            const int units = cur.units - task_unit;                                 // of this task, if less than N
            int place = cur.place + task_unit * KEYS;
            if (place >= ring.keys) place -= ring.keys;
            const bool full = first_key + N * KEYS - 1 <= len - R;                   // every row sees every key
            float* buf = s_sm + (stage & 1) * s_other;
            for (int gq = 0; gq < group; ++gq) {
                float acc[N][PARTS][4];
                need_queries(head0 + gq);
                const bool last = gq == group - 1;
                if (last) more = advance();
                // the loads of the next keys start as soon as their registers are free, one tile after the other
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if constexpr (HALF) {
                        keys[i].template score<NT * 8>(acc[i], lane, [&](int m_, int x) { return q[m_][x]; });
                    } else {
                        const T* qh = queries + (long)(head0 + gq) * c.D;
                        keys[i].template score<NT * 8>(acc[i], lane, [&](int row, int ch) {
                            const long r = q_at[row];
                            const int e = K::element(ch, t4);
                            return r >= 0 && e < c.D ? *reinterpret_cast<const uint4*>(qh + r + e) : make_uint4(0, 0, 0, 0);
                        });
                    }
                    if (last && more) load(i);
                }
                if (last && more) {
                    query_rows();
                    need_queries((cur.hk0 + task_hk) * group);
                }
                float* s = buf + ((local + gq) >> 1) * R * ring.row + ((local + gq) & 1);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (i > 0 && i >= units) break;
                    const int key = first_key + i * KEYS;
                    if (!full) {
#pragma unroll
                        for (int p = 0; p < PARTS; ++p)
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                if (key + K::key_of(p, y, lane) > len - R + K::row_of(p, y, lane)) acc[i][p][y] = 0.0f;
                    }
                    float* to = s + (place + i * KEYS >= ring.keys ? place + i * KEYS - ring.keys : place + i * KEYS);
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            if (HALF && y >= 2 && NT == 1) continue;                 // rows 8 to 15
                            const int row = K::row_of(p, y, lane), kk = K::key_of(p, y, lane);
                            if (row < R) to[row * ring.row + (kk & ~3) + (kk & 1) * 2 + (kk & 2 ? ring.half : 0)] = acc[i][p][y];
                        }
                    }
                }
            }
        }
        // stages behind this warp's last task: the cursor stands behind the run's last stage
        while (stage < cur.stage) {
            barrier_arrive(BAR_FULL + (stage & 1), THREADS);
            ++stage;
            if (stage >= 2 && stage < cur.stage) barrier_sync(BAR_EMPTY + (stage & 1), THREADS);
        }
        return;
    }

    // ---- conv, head mix, softmax statistics
    fewer_registers();
    const int tid = threadIdx.x - ROLE_THREADS;
    load_mix(W_sm, a.W1, H, a.w_dtype);
    for (int i = tid; i < (H + 1) / 2 * a.cq * ckp; i += ROLE_THREADS) {
        const int j = i % ckp - first_tap, row = i / ckp, tap = row % a.cq, h = row / a.cq * 2;
        const long at = ((long)h * a.cq + tap) * a.ck + j;
        t_sm[i + h] = make_float2(j >= 0 && j < a.ck ? load_weight(a.w1, at, a.w_dtype) * a.scale : 0.0f,
                              j >= 0 && j < a.ck && h + 1 < H ? load_weight(a.w1, at + a.cq * a.ck, a.w_dtype) * a.scale : 0.0f);
    }
    const int quads = tile / 4, oquads = round4(H) / 4;
    int stage = 0, stages = 0;                                   // of the whole run: what is not waited for at its end
    for (long x = begin; x < end;) {
        const Span s = span_at(c, before, lens, a.B, x, end);
        stages += (s.k1 - s.k0 + tile - 1) / tile * ((a.score_heads + a.kv_together - 1) / a.kv_together);
        x = (long)before[s.b] + s.k1 / KEYS;
    }
    int turn = 0;
    for (long x = begin; x < end;) {
        const Span s = span_at(c, before, lens, a.B, x, end);
        turn = ring_turn(ring, whole, turn, s.k0 - hl);
        for (int i = tid; i < a.cq2 * H * quads; i += ROLE_THREADS) ml[i] = make_float2(-INFINITY, 0.0f);
        const int limit = s.k1 < s.len ? s.k1 : s.len;           // keys from here on are another run's
        for (int k0 = s.k0; k0 < s.k1; k0 += tile) {
            for (int hk0 = 0; hk0 < a.score_heads; hk0 += a.kv_together, ++stage) {
                barrier_sync(BAR_FULL + (stage & 1), THREADS);
                // conv: (two heads, row, four keys) a thread
                const int heads = (a.score_heads - hk0 < a.kv_together ? a.score_heads - hk0 : a.kv_together) * group;
                const int q0 = ((k0 - left - first_tap + turn + ring.keys) % ring.keys) >> 2;
                const float* s_now = s_sm + (stage & 1) * s_other;
                const float2* t_now = t_sm + hk0 * group / 2 * pair_taps(a.cq, a.ck);
                float* c_now = c_sm + ((hk0 * group) << a.shift);
                switch (ckp / 4) {
                    case 1: conv_pairs<1>(s_now, t_now, c_now, ring, q0, heads, H, R, a.cq, a.cq2, ckp, a.shift, tid); break;
                    case 2: conv_pairs<2>(s_now, t_now, c_now, ring, q0, heads, H, R, a.cq, a.cq2, ckp, a.shift, tid); break;
                    case 3: conv_pairs<3>(s_now, t_now, c_now, ring, q0, heads, H, R, a.cq, a.cq2, ckp, a.shift, tid); break;
                    case 4: conv_pairs<4>(s_now, t_now, c_now, ring, q0, heads, H, R, a.cq, a.cq2, ckp, a.shift, tid); break;
                    default: conv_pairs<0>(s_now, t_now, c_now, ring, q0, heads, H, R, a.cq, a.cq2, ckp, a.shift, tid); break;
                }
                if (stage + 2 < stages) barrier_arrive(BAR_EMPTY + (stage & 1), THREADS);
            }
            barrier_sync(BAR_MATH, ROLE_THREADS);
            // head mix and softmax statistics: (row, four heads, four keys) a thread
            for (int i = tid; i < a.cq2 * oquads << (a.shift - 2); i += ROLE_THREADS) {
                const int kq = (i & (quads - 1)) * 4, rest = i >> (a.shift - 2), r = rest / oquads, o0 = (rest - r * oquads) * 4;
                if (k0 + kq >= limit) continue;
                float z[4][4];
                mix_heads(z, W_sm + o0, c_sm + ((r * H) << a.shift) + kq, H, tile);
                const int seen = s.len - a.cq2 + r - k0 - kq;                        // of the four keys those up to this one are seen by the row
#pragma unroll
                for (int o = 0; o < 4; ++o) {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (k > seen) z[o][k] = -INFINITY;
                    const int row = r * H + o0 + o;
                    if (o0 + o < H) {
                        // maximum and sum of this thread's own keys of the run
                        const float2 old = ml[row * quads + kq / 4];
                        const float top = fmaxf(fmaxf(fmaxf(z[o][0], z[o][1]), fmaxf(z[o][2], z[o][3])), old.x);
                        // while nothing has been seen the maximum is -inf and the sum 0
                        const float ref = top == -INFINITY ? 0.0f : top;
                        float sum = old.y * fast_exp2(old.x - ref);
#pragma unroll
                        for (int k = 0; k < 4; ++k) sum += fast_exp2(z[o][k] - ref);
                        ml[row * quads + kq / 4] = make_float2(top, sum);
                        *reinterpret_cast<float4*>(a.logits + ((long)s.b * a.cq2 * H + row) * a.pitch + k0 + kq) = make_float4(z[o][0], z[o][1], z[o][2], z[o][3]);
                    }
                }
            }
            barrier_sync(BAR_MATH, ROLE_THREADS);                // the next tile's conv writes where this mix reads
        }
        for (int i = tid; i < a.cq2 * H; i += ROLE_THREADS) {
            float top = -INFINITY, sum = 0.0f;
            for (int k = 0; k < quads; ++k) top = fmaxf(top, ml[i * quads + (k + i) % quads].x);
            const float ref = top == -INFINITY ? 0.0f : top;
            for (int k = 0; k < quads; ++k) {
                const float2 v = ml[i * quads + (k + i) % quads];
                sum = fmaf(v.y, fast_exp2(v.x - ref), sum);
            }
            a.part_ml[(me + s.b) * a.cq2 * H + i] = make_float2(top, sum);
        }
        barrier_sync(BAR_MATH, ROLE_THREADS);
        turn += s.k0 + (s.k1 - s.k0 + tile - 1) / tile * tile + hr;                  // the place behind the span's last tile
        x = (long)before[s.b] + s.k1 / KEYS;
    }
}

// Tasks of (GT query heads, share of a tile's keys) belong to one warp each; where heads do not divide evenly among the warps, `copies`
// warps share one and each keeps an output of its own.
template <typename T, int DMAX, int GT>
__global__ void __launch_bounds__(THREADS, 1) mta_decode_values_kernel(PagedCache c, MtaArgs a, int copy_shift) {
    constexpr bool HALF = sizeof(T) == 2;
    using V = std::conditional_t<HALF, ValueTile<T, DMAX>, ValueTileF32<DMAX>>;
    using P = Pieces<GT>;
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int H = c.H, group = H / c.kv_heads, tile = 1 << a.shift, ckp = round4(a.ck2), left = (a.ck2 - 1) / 2, pp = prob_pitch(tile, a.ck2);
    const int quads = tile / 4, oquads = round4(H) / 4, ap = piece_pitch(tile), copies = 1 << copy_shift;
    const ValueSmem m = value_smem(a.B, H, c.D, tile, a.cq2, a.ck2, copies);
    float *p_sm = reinterpret_cast<float*>(smem + m.p), *y_sm = reinterpret_cast<float*>(smem + m.y), *by = reinterpret_cast<float*>(smem + m.by);
    float *W_sm = reinterpret_cast<float*>(smem + m.W), *t_sm = reinterpret_cast<float*>(smem + m.taps), *o_sm = reinterpret_cast<float*>(smem + m.o);
    T* a_sm = reinterpret_cast<T*>(smem + m.a);                  // by the stage's parity: [head][piece][key], float32: [head][key]
    const int a_other = (int)(m.a_one / sizeof(T));
    float *top_sm = reinterpret_cast<float*>(smem + m.ml), *r_sm = reinterpret_cast<float*>(smem + m.run_taps);
    int *before = reinterpret_cast<int*>(smem + m.before), *lens = before + a.B + 1;

    // The lengths, the tables, the values and the weights are not written by the kernel before.
    count_tiles(c, a.B, 4, before, lens);
    __syncthreads();
    const long n = before[a.B], workers = n < a.workers ? n : a.workers, me = blockIdx.x;
    if (me >= workers) return;
    const long begin = run_begin(me, n, workers), end = run_begin(me + 1, n, workers);

    if (warp >= ROLE_WARPS) {
        // ---- product with the values.  A stage is a tile; the loads run ahead of the arithmetic as in the scores kernel.
        more_registers();
        const int tid = threadIdx.x - ROLE_THREADS, me_warp = warp - ROLE_WARPS, tasks = H / GT * copies;
        const T* pool = static_cast<const T*>(c.v);
        const int head_stride = c.D << c.page_shift;
        struct Cursor {
            Span s;
            long at;
            int k0, units, task, unit, last, stage;
            long head;         // from kv head 0 to the task's
            Pages next;
            bool done;
        } cur = {};
        // The units of this stage that the task's copy has, and where its kv head lies.  Divisions by the group only where they must be: in
        // the stream of loads they cost more than the products.
        auto share = [&] {
            const int copy = cur.task & (copies - 1), all = tile / KEYS, h = cur.task >> copy_shift;
            cur.unit = copy * all >> copy_shift;
            cur.last = (copy + 1) * all >> copy_shift;
            if (cur.last > cur.units) cur.last = cur.units;
            cur.head = (long)(group == GT ? h : h * GT / group) * head_stride;
        };
        auto enter_stage = [&] {
            cur.units = ((cur.k0 + tile < cur.s.k1 ? cur.k0 + tile : cur.s.k1) - cur.k0) / KEYS;
            const int key = cur.k0 + lane * KEYS;
            const bool on = lane < cur.units && key < cur.s.len;
            if (cur.k0 == cur.s.k0) cur.next.look_up(c, cur.s.slot, key, on);
            cur.at = cur.next.at(c, key, on);
            const bool ahead = lane < tile / KEYS && key + tile < cur.s.len;
            cur.next.look_up(c, cur.s.slot, key + tile, ahead);
            cur.task = me_warp;
            share();
        };
        auto enter_span = [&](long x) {
            cur.s = span_at(c, before, lens, a.B, x, end);
            cur.k0 = cur.s.k0;
        };
        enter_span(begin);
        enter_stage();
        constexpr int N = TOGETHER<T, DMAX>;
        V values[N];
        int t_task = 0, t_unit = 0, t_units = 0, next_live = 0;  // whose values are on their way or next
        long next_at[N];
        bool t_first = false;                                    // of its task and stage
        auto advance = [&]() -> bool {
            while (!cur.done && (cur.task >= tasks || cur.unit >= cur.last)) {
                if (cur.task < tasks) {
                    cur.task += ROLE_WARPS;
                    if (cur.task < tasks) share();
                    continue;
                }
                ++cur.stage;
                cur.k0 += tile;
                if (cur.k0 >= cur.s.k1) {
                    const long x = (long)before[cur.s.b] + cur.s.k1 / KEYS;
                    if (x >= end) { cur.done = true; break; }
                    enter_span(x);
                }
                enter_stage();
            }
            if (cur.done) return false;
            const int copy = cur.task & (copies - 1);
            const long head = cur.head;
            t_task = cur.task; t_unit = cur.unit;
            t_first = cur.unit == copy * (tile / KEYS) >> copy_shift;
            t_units = cur.last - cur.unit;                       // N or fewer: the last of the task and stage
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const long base = __shfl_sync(0xffffffffu, cur.at, cur.unit + i);
                next_at[i] = base < 0 ? base : base + head;
            }
            next_live = cur.s.len - (cur.k0 + cur.unit * KEYS);
            cur.unit += N;
            return true;
        };
        auto load = [&](int i) {
            if (i == 0 || i < t_units) values[i].load(pool, next_at[i], next_live - i * KEYS, c.D, lane);
        };
        int stage = 0, stages = 0;
        for (long x = begin; x < end;) {
            const Span s = span_at(c, before, lens, a.B, x, end);
            stages += (s.k1 - s.k0 + tile - 1) / tile;
            x = (long)before[s.b] + s.k1 / KEYS;
        }
        for (int i = tid; i < copies * H * c.D; i += ROLE_THREADS) o_sm[i] = 0.0f;
        constexpr int CH = HALF ? DMAX / 64 : 1;
        float acc[HALF ? CH : GT][4][4];                         // mma accumulators; float32: [head][0][element]
        // The outputs of a span, once all of this half are done with it.
        auto put_out = [&](int b) {
            barrier_sync(BAR_MEMORY, ROLE_THREADS);
            const long u0 = before[b], u1 = before[b + 1];
            const bool only = run_owner(u0, n, workers) == run_owner(u1 - 1, n, workers);
            for (int i = tid; i < H * c.D; i += ROLE_THREADS) {
                float v = 0.0f;
                for (int y = 0; y < copies; ++y) {
                    v += o_sm[y * H * c.D + i];
                    o_sm[y * H * c.D + i] = 0.0f;
                }
                if (only) static_cast<T*>(a.out)[(long)b * H * c.D + i] = from_f32<T>(v);      // the only run of the sequence
                else a.part_o[(me + b) * H * c.D + i] = v;
            }
            barrier_sync(BAR_MEMORY, ROLE_THREADS);
        };
        // Every warp of this half passes every stage, with or without a task in it, and the ends of spans between them, so that all meet
        // the same barriers in the same order.
        long span_x = begin;
        Span span = span_at(c, before, lens, a.B, begin, end);
        int span_end = (span.k1 - span.k0 + tile - 1) / tile;    // the stage behind the span's last
        auto pass_stages = [&](int to) {
            while (stage < to) {
                if (stage + 2 < stages) barrier_arrive(BAR_EMPTY + (stage & 1), THREADS);
                if (++stage == span_end) {
                    put_out(span.b);
                    span_x = (long)before[span.b] + span.k1 / KEYS;
                    if (span_x < end) {
                        span = span_at(c, before, lens, a.B, span_x, end);
                        span_end += (span.k1 - span.k0 + tile - 1) / tile;
                    }
                }
                if (stage < stages) barrier_sync(BAR_FULL + (stage & 1), THREADS);
            }
        };
        barrier_sync(BAR_MEMORY, ROLE_THREADS);                  // the outputs are zero
        bool started = false;
        bool more = advance();
        if (more) {
#pragma unroll
            for (int i = 0; i < N; ++i) load(i);
        }
        while (more) {
            // the cursor still stands where this task's values lie
            if (!started) barrier_sync(BAR_FULL, THREADS);       // the first stage
            started = true;
            pass_stages(cur.stage);
            const int unit = t_unit, units = t_units, copy = t_task & (copies - 1), h0 = (t_task >> copy_shift) * GT;
            const bool first = t_first, final = t_units <= N;
            const T* weights = a_sm + (stage & 1) * a_other;
            if (first) {
#pragma unroll
                for (int i = 0; i < (HALF ? CH : GT); ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.0f;
            }
            if constexpr (HALF) {
                const int y = g / P::STRIDE, column = g % P::STRIDE;
                const bool on = y < GT && column < P::WIDTH;
                const uint32_t* col[P::SETS];
#pragma unroll
                for (int s = 0; s < P::SETS; ++s)
                    col[s] = reinterpret_cast<const uint32_t*>(weights + (on ? ((h0 + y) * P::PIECES + P::piece_of(s, column)) * ap : 0)) + t4 + unit * 8;
                more = advance();
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    if (i == 0 || i < units) {
                        uint32_t w[P::SETS][2];
#pragma unroll
                        for (int s = 0; s < P::SETS; ++s) {
                            w[s][0] = on ? col[s][i * 8] : 0u;
                            w[s][1] = on ? col[s][i * 8 + 4] : 0u;
                        }
                        values[i].multiply(acc, w);
                    }
                    if (more) load(i);
                }
                if (final) {
                    // sum over the pieces; a head's columns are those of one lane (four heads) or of two, which then halve the elements
                    const int head = h0 + t4 * 2 / P::STRIDE;
                    const bool mine = t4 * 2 / P::STRIDE < GT;
                    float* to = o_sm + (copy * H + (mine ? head : 0)) * c.D;
                    const float back = std::is_same_v<T, __half> && mine ? 1.0f / by[head] : 1.0f;
#pragma unroll
                    for (int i = 0; i < CH; ++i) {
                        float f[P::SUMS];
                        P::sum_columns(f, acc[i], t4);
                        const int e0 = V::element(i, g) + (P::STRIDE == 4 ? (t4 & 1) * 4 : 0);
                        if (!mine || V::element(i, g) >= c.D) continue;
#pragma unroll
                        for (int e = 0; e < P::SUMS; e += 4) {
                            float4* at = reinterpret_cast<float4*>(to + e0 + e);
                            float4 v = *at;
                            v.x = fmaf(f[e], back, v.x); v.y = fmaf(f[e + 1], back, v.y); v.z = fmaf(f[e + 2], back, v.z); v.w = fmaf(f[e + 3], back, v.w);
                            *at = v;
                        }
                    }
                }
            } else {
#pragma unroll
                for (int n_ = 0; n_ < N; ++n_) {
                    if (n_ > 0 && n_ >= units) break;
#pragma unroll
                    for (int i = 0; i < V::STEPS; ++i) {
                        float f[4];
                        unpack16(values[n_].r[i], f);
#pragma unroll
                        for (int y = 0; y < GT; ++y) {
                            const float p = weights[((h0 + y) << a.shift) + (unit + n_) * KEYS + i * V::SUBS + lane / V::ROWLANES];
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[y][0][e] = fmaf(p, f[e], acc[y][0][e]);
                        }
                    }
                }
                more = advance();
                if (more) {
#pragma unroll
                    for (int i = 0; i < N; ++i) load(i);
                }
                if (final) {
                    const int e0 = (lane % V::ROWLANES) * 4;
#pragma unroll
                    for (int y = 0; y < GT; ++y) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
#pragma unroll
                            for (int s = V::ROWLANES; s < 32; s <<= 1) acc[y][0][e] += __shfl_xor_sync(0xffffffffu, acc[y][0][e], s);
                        if (lane < V::ROWLANES && e0 < c.D) {
                            float4* at = reinterpret_cast<float4*>(o_sm + (copy * H + h0 + y) * c.D + e0);
                            float4 v = *at;
                            v.x += acc[y][0][0]; v.y += acc[y][0][1]; v.z += acc[y][0][2]; v.w += acc[y][0][3];
                            *at = v;
                        }
                    }
                }
            }
        }
        if (!started) barrier_sync(BAR_FULL, THREADS);           // no task at all
        pass_stages(stages);
        return;
    }

    // ---- probabilities, conv, head mix: the weights of the values
    fewer_registers();
    const int tid = threadIdx.x;
    load_mix(W_sm, a.W2, H, a.w_dtype);
    for (int i = tid; i < H * a.cq2 * ckp; i += ROLE_THREADS) {
        const int j = i % ckp, row = i / ckp;
        t_sm[i] = j < a.ck2 ? load_weight(a.w2, (long)row * a.ck2 + j, a.w_dtype) : 0.0f;
    }
    barrier_sync(BAR_MATH, ROLE_THREADS);
    if constexpr (std::is_same_v<T, __half>) {
        // Probabilities are at most 1, so a weight of head o is at most A = sum_h |W2[o,h]| sum |w2[h]|.  Times 2^14 over the power of two
        // below A it stays under 2^15.  Its three pieces are normal numbers of fp16, and add up to it within 2^-33 of it, only while it is above
        // about 2^-6 A (the first alone down to 2^-28 A); below that the last of them is off by half of fp16's smallest number, 2^-39 A.
        for (int h = tid; h < H; h += ROLE_THREADS) {
            float s = 0.0f;
            for (int i = 0; i < a.cq2 * ckp; ++i) s += fabsf(t_sm[h * a.cq2 * ckp + i]);
            y_sm[h] = s;
        }
        barrier_sync(BAR_MATH, ROLE_THREADS);
        for (int o = tid; o < H; o += ROLE_THREADS) {
            float s = 0.0f;
            for (int h = 0; h < H; ++h) s = fmaf(fabsf(W_sm[h * round4(H) + o]), y_sm[h], s);
            by[o] = s > 1e-30f && s < 1e30f ? exp2f((float)(14 - ilogbf(s))) : 1.0f;
        }
        barrier_sync(BAR_MATH, ROLE_THREADS);
    }
    pdl_wait();
    int stage = 0;
    for (long x = begin; x < end;) {
        const Span s = span_at(c, before, lens, a.B, x, end);
        const long w0 = run_owner(before[s.b], n, workers), w1 = run_owner((long)before[s.b + 1] - 1, n, workers);
        // maximum and one over the sum of every (row, head), from all runs of the sequence: eight lanes each
        for (int i0 = tid / 8; i0 < (a.cq2 * H + 31) / 32 * 32; i0 += ROLE_THREADS / 8) {
            const int i = i0 < a.cq2 * H ? i0 : a.cq2 * H - 1;
            const float2* parts = a.part_ml + (long)s.b * a.cq2 * H + i;
            float top = -INFINITY, sum = 0.0f;
            for (long w = w0 + tid % 8; w <= w1; w += 32) {
                float2 v[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) v[y] = w + 8 * y <= w1 ? parts[(w + 8 * y) * a.cq2 * H] : make_float2(-INFINITY, 0.0f);
                const float t = fmaxf(fmaxf(fmaxf(v[0].x, v[1].x), fmaxf(v[2].x, v[3].x)), top), ref = t == -INFINITY ? 0.0f : t;
                sum *= fast_exp2(top - ref);
#pragma unroll
                for (int y = 0; y < 4; ++y) sum = fmaf(v[y].y, fast_exp2(v[y].x - ref), sum);
                top = t;
            }
#pragma unroll
            for (int y = 1; y < 8; y <<= 1) {
                const float v = __shfl_xor_sync(0xffffffffu, top, y), l = __shfl_xor_sync(0xffffffffu, sum, y);
                const float t = fmaxf(top, v), ref = t == -INFINITY ? 0.0f : t;
                sum = sum * fast_exp2(top - ref) + l * fast_exp2(v - ref);
                top = t;
            }
            // the conv's taps of this sequence have the sums in them; a row before the first token has no keys: its probabilities are zero
            const int row = i / H, h = i - row * H;
            const float over = s.len - a.cq2 + row < 0 ? 0.0f : 1.0f / sum;
            if (i0 < a.cq2 * H) {
                if (tid % 8 == 0) top_sm[i] = s.len - a.cq2 + row < 0 ? 0.0f : top;
                for (int j = tid % 8; j < ckp; j += 8) r_sm[(h * a.cq2 + row) * ckp + j] = t_sm[(h * a.cq2 + row) * ckp + j] * over;
            }
        }
        barrier_sync(BAR_MATH, ROLE_THREADS);
        const int limit = s.k1 < s.len ? s.k1 : s.len;
        for (int k0 = s.k0; k0 < s.k1; k0 += tile, ++stage) {
            // exponentials (the taps hold one over their sums), then those of the neighbours' keys that the conv reaches
            const float* logits = a.logits + (long)s.b * a.cq2 * H * a.pitch + k0;
#pragma unroll 4
            for (int i = tid; i < a.cq2 * H << (a.shift - 2); i += ROLE_THREADS) {
                const int row = i >> (a.shift - 2), kq = (i & (quads - 1)) * 4;
                const float top = top_sm[row];
                float4 z = make_float4(0, 0, 0, 0);
                if (k0 + kq < s.len) z = *reinterpret_cast<const float4*>(logits + row * a.pitch + kq);
                const float e[4] = {z.x, z.y, z.z, z.w};
                float* p = p_sm + row * pp + left + kq;
#pragma unroll
                for (int k = 0; k < 4; ++k) p[k] = k0 + kq + k < s.len ? fast_exp2(e[k] - top) : 0.0f;
            }
            const int beside = pp - tile;
#pragma unroll 2
            for (int i = tid; i < a.cq2 * H * beside; i += ROLE_THREADS) {
                const int row = i / beside, x_ = i - row * beside, col = x_ < left ? x_ : x_ + tile, key = k0 - left + col;
                p_sm[row * pp + col] = key >= 0 && key < s.len && col < tile + a.ck2 - 1 ? fast_exp2(logits[row * a.pitch + key - k0] - top_sm[row]) : 0.0f;
            }
            barrier_sync(BAR_MATH, ROLE_THREADS);
            for (int i = tid; i < H << (a.shift - 2); i += ROLE_THREADS) {
                const int quad = i & (quads - 1), h = i >> (a.shift - 2);
                float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                for (int tap = 0; tap < a.cq2; ++tap) conv_row(z, p_sm + (tap * H + h) * pp + 4 * quad, r_sm + (h * a.cq2 + tap) * ckp, ckp);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k0 + 4 * quad + e >= limit) z[e] = 0.0f;
                *reinterpret_cast<float4*>(y_sm + (h << a.shift) + 4 * quad) = make_float4(z[0], z[1], z[2], z[3]);
            }
            barrier_sync(BAR_MATH, ROLE_THREADS);
            if (stage >= 2) barrier_sync(BAR_EMPTY + (stage & 1), THREADS);
            T* to = a_sm + (stage & 1) * a_other;
            for (int i = tid; i < oquads << (a.shift - 2); i += ROLE_THREADS) {
                const int kq = (i & (quads - 1)) * 4, o0 = (i >> (a.shift - 2)) * 4;
                float z[4][4];
                mix_heads(z, W_sm + o0, y_sm + kq, H, tile);
#pragma unroll
                for (int o = 0; o < 4; ++o) {
                    if (o0 + o >= H) break;
                    if constexpr (HALF) {
                        float f[4][P::PIECES];
#pragma unroll
                        for (int k = 0; k < 4; ++k) split_pieces<T, P::SETS>(std::is_same_v<T, __half> ? z[o][k] * by[o0 + o] : z[o][k], f[k]);
#pragma unroll
                        for (int piece = 0; piece < P::PIECES; ++piece)
                            *reinterpret_cast<uint2*>(to + ((o0 + o) * P::PIECES + piece) * ap + kq) =
                                make_uint2(pack2<T>(f[0][piece], f[1][piece]), pack2<T>(f[2][piece], f[3][piece]));
                    } else {
                        *reinterpret_cast<float4*>(to + ((o0 + o) << a.shift) + kq) = make_float4(z[o][0], z[o][1], z[o][2], z[o][3]);
                    }
                }
            }
            barrier_arrive(BAR_FULL + (stage & 1), THREADS);
        }
        x = (long)before[s.b] + s.k1 / KEYS;
    }
}

// One block per (head, sequence): adds the runs' outputs in the order of their keys.  Sequences of no tokens get zeros.
template <typename T> __global__ void __launch_bounds__(128) mta_decode_join_kernel(PagedCache c, MtaArgs a) {
    extern __shared__ __align__(16) char smem[];
    int *before = reinterpret_cast<int*>(smem), *lens = before + a.B + 1;
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
    int shift, split, kv_together, gt, copies, workers;
    size_t score_bytes, value_bytes;               // shared memory
    size_t ml_at, o_at, bytes;                     // workspace
    long pitch;
};

int make_plan(Plan* p, int B, int H, int kv_heads, int D, int cq, int ck, int cq2, int ck2, int max_length) {
    const int group = H / kv_heads;
    p->gt = group % 4 == 0 ? 4 : group % 2 == 0 ? 2 : 1;
    const long units = (long)B * ((max_length + KEYS - 1) / KEYS);
    p->workers = (int)(units < DECODE_SMS ? (units < 1 ? 1 : units) : DECODE_SMS);
    // tiles of 64 keys, or as many as the longest run has: 19 runs of 16 keys 29.3 us with tiles of 64, 26.7 with tiles of 16; runs of 155
    // keys 80 us with tiles of 64, 82 with 32, 101 with 16
    int shift = 6;
    const long run = (units + p->workers - 1) / p->workers * KEYS;
    while (shift > 4 && 1L << (shift - 1) >= run) --shift;
    bool fits = false;
    for (p->shift = shift; p->shift >= 4 && !fits; --p->shift) {
        const int tile = 1 << p->shift;
        // shares of a tile's units: the fewest that leave the warps least idle
        p->copies = 1;
        auto rounds = [&](int copies) { return (float)((H / p->gt * copies + ROLE_WARPS - 1) / ROLE_WARPS) / copies; };
        for (int copies = 2; copies <= tile / KEYS; copies *= 2)
            if (rounds(copies) < rounds(p->copies)) p->copies = copies;
        p->value_bytes = value_smem(B, H, D, tile, cq2, ck2, p->copies).bytes;
        // A smaller tile before the heads are taken in parts (of whole pairs), parts of whole groups before parts of a group: every part reads
        // its keys again.
        const int splits = p->shift == 4 ? group : 1;
        for (p->split = 1; p->split <= splits && !fits; ++p->split) {
            if (group % p->split) continue;
            const int heads = kv_heads * p->split, each = group / p->split;
            for (p->kv_together = heads; p->kv_together >= (p->shift == 4 ? 1 : heads) && !fits; --p->kv_together) {
                if (p->kv_together < heads && p->kv_together * each % 2) continue;
                p->score_bytes = score_smem(B, H, each, heads, p->kv_together, tile, cq, ck, cq2).bytes;
                fits = p->score_bytes <= SMEM_MOST && p->value_bytes <= SMEM_MOST;
                if (fits) break;
            }
            if (fits) break;
        }
        if (fits) break;
    }
    MTA_REQUIRE(fits, "mta_decode: %d heads of %d elements with kernels %dx%d and %dx%d need %zu and %zu bytes of shared memory, more than %zu", H, D, cq, ck,
                cq2, ck2, p->score_bytes, value_smem(B, H, D, 16, cq2, ck2, p->copies).bytes, SMEM_MOST);
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
    if (p.gt == 4) rc = launch_kernel<mta_decode_values_kernel<T, DMAX, 4>>("mta_decode_values_kernel", dim3(p.workers), THREADS, p.value_bytes, st, c, a, p.copies == 4 ? 2 : p.copies - 1);
    else if (p.gt == 2) rc = launch_kernel<mta_decode_values_kernel<T, DMAX, 2>>("mta_decode_values_kernel", dim3(p.workers), THREADS, p.value_bytes, st, c, a, p.copies == 4 ? 2 : p.copies - 1);
    else rc = launch_kernel<mta_decode_values_kernel<T, DMAX, 1>>("mta_decode_values_kernel", dim3(p.workers), THREADS, p.value_bytes, st, c, a, p.copies == 4 ? 2 : p.copies - 1);
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
    a.workers = p.workers; a.shift = p.shift; a.score_heads = c.kv_heads * p.split; a.kv_together = p.kv_together;
    // h / split without a division in the stream of loads: h and split are at most 128, so h * (floor(2^16 / split) + 1) exceeds
    // h * 2^16 / split by at most h < 2^16 / split
    a.per_split = 65536 / p.split + 1;
    if (dtype == MTA_F32) return launch<float>(c, a, p, st);
    return dtype == MTA_BF16 ? launch<__nv_bfloat16>(c, a, p, st) : launch<__half>(c, a, p, st);
}

}  // namespace mta
