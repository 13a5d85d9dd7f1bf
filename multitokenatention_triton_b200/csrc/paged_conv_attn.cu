// Conv attention of one new token per sequence over a paged cache:
//
//   s[i,k] = q[t-cq+1+i] . k[k] for k <= t-cq+1+i, else 0      (the last cq queries; t is the newest token)
//   c[k]   = sum_{i,j} w[h,i,j] s[i, k+j-(ck-1)/2]             k <= t
//   out    = sum_k softmax_k(scale * c[k]) v[k]
//
// Every key and value of a head is read once, for cq <= 8 about 2 D cq + 2 cq ck + 2 D = 1.9 kflop per 512 bytes at 6x11 taps and
// D 128: HBM bounds it, and what matters is that enough loads are in flight at every moment.  So a warp works alone, with no
// block-wide barrier: it walks a run of tiles of 16 keys; the scores of a tile are one mma.sync chain (keys are the rows, queries
// the columns) into a ring of three tiles in shared memory, the conv of the tile before it reads that ring, its sixteen logits
// enter a running softmax (maximum, sum and output in float32 registers), and the loads of the next keys and values are issued
// as soon as the registers of the last ones are free.  Runs are equal cuts of all tiles of all sequences and heads, so lengths need
// not be alike; a second kernel joins the runs of a head.
#include "paged.cuh"

namespace mta {
namespace {

constexpr int WARPS = 4;
constexpr int RING = 3 * KEYS, RING_PITCH = RING + 4;   // the pitch spreads an accumulator's rows over the banks

struct ConvAttnArgs {
    const void* w;
    void* out;
    float* part_o;         // (runs' parts, GT, D)
    float2* part_ml;       // (runs' parts, GT): maximum and sum
    int w_dtype, B, cq, ck;
    float scale;           // softmax scale * log2(e): the softmax runs in base 2
    int workers, min_tiles;
};

// Workers that have tiles when there are n tiles: a run is at least min_tiles long.
__device__ __forceinline__ long workers_of(const ConvAttnArgs& a, long n) {
    const long most = (n + a.min_tiles - 1) / a.min_tiles;
    return most < a.workers ? most : a.workers;
}

// GT query heads that share a kv head, NT * 8 >= GT * cq rows of scores.
template <typename T, int DMAX, int GT, int NT> constexpr size_t conv_attn_warp_smem(int cq, int ck) {
    return (size_t)NT * 8 * (DMAX * sizeof(T) + 64) + (size_t)NT * 8 * RING_PITCH * 4 + (size_t)GT * cq * ((ck + 3) / 4 * 4) * 4 + GT * KEYS * 4;
}

template <typename T, int DMAX, int GT, int NT>
__global__ void __launch_bounds__(WARPS * 32, sizeof(T) * DMAX > 256 ? 2 : 4) conv_attn_decode_kernel(PagedCache c, ConvAttnArgs a) {
    using K = KeyTile<T, DMAX>;
    using V = ValueTile<T, DMAX>;
    constexpr int EPL = K::EPL;
    extern __shared__ __align__(16) char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    const int ckp = (a.ck + 3) / 4 * 4;
    char* mine = smem + warp * conv_attn_warp_smem<T, DMAX, GT, NT>(a.cq, a.ck);
    // row pitch of the queries: 64 bytes more than a multiple of 128, so that rows g and g + 1 of an 8-lane phase miss each other's banks
    constexpr int QP = DMAX * (int)sizeof(T) + 64;
    char* q_sm = mine;
    float* s_sm = reinterpret_cast<float*>(mine + NT * 8 * QP);
    float* w_sm = s_sm + NT * 8 * RING_PITCH;
    float* p_sm = w_sm + GT * a.cq * ckp;
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
    const int left = (a.ck - 1) / 2, shift = left & 3;               // `shift` puts a tile's first window on a 16-byte boundary

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

        // queries and taps of this line
        for (int i = lane; i < NT * 8 * (DMAX / EPL); i += 32) {
            const int row = i / (DMAX / EPL), e = (i % (DMAX / EPL)) * EPL, gq = row / a.cq, pos = len - a.cq + row % a.cq;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (gq < GT && pos >= 0 && e < c.D)
                u = *reinterpret_cast<const uint4*>(static_cast<const T*>(c.q_hist) + (((long)slot * c.ring + pos % c.ring) * c.H + h0 + gq) * c.D + e);
            *reinterpret_cast<uint4*>(q_sm + row * QP + e * (int)sizeof(T)) = u;
        }
        for (int i = lane; i < GT * a.cq * ckp; i += 32) {
            const int j = i % ckp, row = i / ckp;
            w_sm[i] = j < a.ck ? load_weight(a.w, ((long)h0 * a.cq + row) * a.ck + j, a.w_dtype) : 0.0f;
        }
        __syncwarp();

        float m[GT], l[GT], o[GT][EPL];
#pragma unroll
        for (int y = 0; y < GT; ++y) {
            m[y] = -INFINITY; l[y] = 0.0f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) o[y][e] = 0.0f;
        }
        K keys;
        V values;
        auto live = [&](int u) { const int r = len - u * KEYS; return r < KEYS ? r : KEYS; };
        auto key_base = [&](int u) { return u >= 0 && u < tiles ? c.at(slot, kv_head, u * KEYS) : -1L; };
        keys.load(k_pool, key_base(u0 - 1), KEYS, c.D, lane);        // a tile before this one is whole
        values.load(v_pool, key_base(u0), live(u0), c.D, lane);
        for (int u = u0 - 1; u <= u1; ++u) {
            float acc[NT][4];
            keys.template score<NT>(acc, lane, [&](int row, int ch) {
                return *reinterpret_cast<const uint4*>(q_sm + row * QP + ch * 64 + t4 * 16);
            });
            if (u < u1) keys.load(k_pool, key_base(u + 1), live(u + 1), c.D, lane);
            const int col = ((u + 3) % 3) * KEYS + shift;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const int row = 8 * nt + 2 * t4 + (y & 1), kk = g + 8 * (y >> 1), key = u * KEYS + kk;
                    // scores above the diagonal are zero; those of tiles outside the sequence are zero already
                    const float s = key <= len - a.cq + row % a.cq ? acc[nt][y] : 0.0f;
                    const int at = col + kk;
                    s_sm[row * RING_PITCH + (at >= RING ? at - RING : at)] = s;
                }
            }
            __syncwarp();
            if (u > u0) {
                const int un = u - 1;
                // conv: lane (i, quad) sums tap rows i, i + 8, ... for four keys, then the eight rows are added
#pragma unroll
                for (int y = 0; y < GT; ++y) {
                    float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    int first = (un % 3) * KEYS + 4 * t4 + shift - left;           // a multiple of 4
                    if (first < 0) first += RING;
                    for (int i = g; i < a.cq; i += 8) {
                        const float4* srow = reinterpret_cast<const float4*>(s_sm + (y * a.cq + i) * RING_PITCH);
                        const float4* wrow = reinterpret_cast<const float4*>(w_sm + (y * a.cq + i) * ckp);
                        int at = first / 4;
                        float4 lo = srow[at];
                        for (int j = 0; j < ckp / 4; ++j) {
                            at = at + 1 == RING / 4 ? 0 : at + 1;
                            const float4 hi = srow[at], w = wrow[j];
                            z[0] = fmaf(w.x, lo.x, fmaf(w.y, lo.y, fmaf(w.z, lo.z, fmaf(w.w, lo.w, z[0]))));
                            z[1] = fmaf(w.x, lo.y, fmaf(w.y, lo.z, fmaf(w.z, lo.w, fmaf(w.w, hi.x, z[1]))));
                            z[2] = fmaf(w.x, lo.z, fmaf(w.y, lo.w, fmaf(w.z, hi.x, fmaf(w.w, hi.y, z[2]))));
                            z[3] = fmaf(w.x, lo.w, fmaf(w.y, hi.x, fmaf(w.z, hi.y, fmaf(w.w, hi.z, z[3]))));
                            lo = hi;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
#pragma unroll
                        for (int s = 4; s < 32; s <<= 1) z[e] += __shfl_xor_sync(0xffffffffu, z[e], s);
                        z[e] = un * KEYS + 4 * t4 + e < len ? z[e] * a.scale : -INFINITY;
                    }
                    float top = fmaxf(fmaxf(z[0], z[1]), fmaxf(z[2], z[3]));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const float m_new = fmaxf(m[y], top);
                    // while every logit so far is -inf nothing has been summed: a finite stand-in keeps -inf - -inf away
                    const float ref = m_new == -INFINITY ? 0.0f : m_new;
                    const float fade = exp2f(m[y] - ref);
                    float sum = 0.0f, p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) { p[e] = exp2f(z[e] - ref); sum += p[e]; }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    l[y] = l[y] * fade + sum;
                    m[y] = m_new;
#pragma unroll
                    for (int e = 0; e < EPL; ++e) o[y][e] *= fade;
                    if (g == 0) *reinterpret_cast<float4*>(p_sm + y * KEYS + 4 * t4) = make_float4(p[0], p[1], p[2], p[3]);
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < V::STEPS; ++i) {
                    float f[EPL];
                    unpack16<T>(values.r[i], f);
#pragma unroll
                    for (int y = 0; y < GT; ++y) {
                        const float p = p_sm[y * KEYS + i * V::SUBS + lane / V::ROWLANES];
#pragma unroll
                        for (int e = 0; e < EPL; ++e) o[y][e] = fmaf(p, f[e], o[y][e]);
                    }
                }
                if (u < u1) values.load(v_pool, key_base(u), live(u), c.D, lane);
            }
            __syncwarp();
        }
#pragma unroll
        for (int y = 0; y < GT; ++y)
#pragma unroll
            for (int e = 0; e < EPL; ++e)
#pragma unroll
                for (int s = V::ROWLANES; s < 32; s <<= 1) o[y][e] += __shfl_xor_sync(0xffffffffu, o[y][e], s);
        const int e0 = (lane % V::ROWLANES) * EPL;
        if (lane < V::ROWLANES && e0 < c.D) {
            if (u0 == 0 && u1 == tiles) {                            // the whole line: nothing to join
#pragma unroll
                for (int y = 0; y < GT; ++y) {
#pragma unroll
                    for (int e = 0; e < EPL; ++e) o[y][e] /= l[y];
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + ((long)b * c.H + h0 + y) * c.D + e0) = pack16<T>(o[y]);
                }
            } else {
                const long part = me + (long)b * lines + line;
#pragma unroll
                for (int y = 0; y < GT; ++y) {
                    float* to = a.part_o + (part * GT + y) * c.D + e0;
#pragma unroll
                    for (int e = 0; e < EPL; e += 4) *reinterpret_cast<float4*>(to + e) = make_float4(o[y][e], o[y][e + 1], o[y][e + 2], o[y][e + 3]);
                    if (lane == 0) a.part_ml[part * GT + y] = make_float2(m[y], l[y]);
                }
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

constexpr int MIN_TILES = 4;

// Query heads that a warp takes together: all that share a kv head if the scores of at most four fit in 32 rows.
int heads_together(int group, int cq) {
    if (group % 4 == 0 && 4 * cq <= DECODE_MAX_ROWS) return 4;
    if (group % 2 == 0 && 2 * cq <= DECODE_MAX_ROWS) return 2;
    return 1;
}

struct Plan {
    int gt, workers;
    size_t ml_bytes, bytes;
};

Plan make_plan(int B, int H, int kv_heads, int D, int cq, int max_length) {
    Plan plan, *p = &plan;
    p->gt = heads_together(H / kv_heads, cq);
    const long lines = (long)B * (H / p->gt), tiles = lines * ((max_length + KEYS - 1) / KEYS);
    long workers = (tiles + MIN_TILES - 1) / MIN_TILES;
    const long most = (long)DECODE_SMS * 16;
    p->workers = (int)(workers < most ? (workers < 1 ? 1 : workers) : most);
    const size_t parts = (size_t)(p->workers + lines) * p->gt;
    p->ml_bytes = (parts * sizeof(float2) + 255) / 256 * 256;
    p->bytes = p->ml_bytes + parts * D * sizeof(float);
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
    const int nt = (gt * a.cq + 7) / 8;
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
    return make_plan(B, H, kv_heads, D, cq, max_length).bytes;
}

int conv_attn_decode_launch(const PagedCache& cache, const void* w, int w_dtype, void* out, void* workspace, int B, int cq, int ck, float scale, int dtype,
                            cudaStream_t st) {
    PagedCache c = cache;
    if (int rc = wait_flag_ptr(&c.err)) return rc;
    const Plan p = make_plan(B, c.H, c.kv_heads, c.D, cq, c.max_length);
    ConvAttnArgs a;
    a.w = w; a.w_dtype = w_dtype; a.out = out; a.B = B; a.cq = cq; a.ck = ck; a.scale = scale * LOG2E;
    a.part_ml = static_cast<float2*>(workspace);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.ml_bytes);
    a.workers = p.workers; a.min_tiles = MIN_TILES;
    if (dtype == MTA_F32) return launch_dim<float>(c, a, p.gt, st);
    return dtype == MTA_BF16 ? launch_dim<__nv_bfloat16>(c, a, p.gt, st) : launch_dim<__half>(c, a, p.gt, st);
}

}  // namespace mta
