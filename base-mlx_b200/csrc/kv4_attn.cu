// Attention over the 4-bit KV cache, optionally accumulating each key's
// attention weight.
//
// Row i of sequence b (n_b new rows behind off_b cached positions, T_b = off_b +
// n_b) and query head h see the keys j < T_b of kv head h / G, with `causal`
// only j <= off_b + i:
//   s_j = scale <q, k_j>, lse = log sum_j exp(s_j), out = sum_j exp(s_j - lse) v_j,
//   mass[b][kv head][j] += sum over the rows and the kv head's query heads of exp(s_j - lse).
// A row that sees no key (a row past n_b, or an empty sequence) gives out = 0, lse = -inf.
//
// A column is one (row, query head) of a kv head: column c = i G + head.  The
// work of a call is the list of (sequence, kv head, column block) segments,
// each of ceil(T_b / 32) tiles of 32 keys; the thread blocks take equal
// contiguous shares of that list, whatever the lengths, so a ragged batch and
// one long sequence both fill the GPU.  A segment inside one share is finished
// there; one that spans shares leaves a partial (base exponent, sum, output) per
// share, which a second kernel joins.  Caches so short that a cluster of blocks
// holds a segment in a few tiles per warp skip the list and join in the cluster.
#include <algorithm>

#include "kv4_join.cuh"
#include "kv4_launch.h"
#include "kv4_tc.h"
#include "kv4_tile.cuh"
#include "smem_attr.h"

namespace qw {
namespace {

using namespace kv4;

constexpr int AW = 8, ANT = 32 * AW;  // warps and threads of a block
constexpr int ASTAGES = 3;            // tiles of a warp's load ring
constexpr int MAX_CLUSTER = 8;

QW_DEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// The pair (four) of floats at `p` in the cluster's block `rank`.
QW_DEV float2 cluster_load2(const float* p, int rank) {
    uint32_t addr;
    float2 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
    return v;
}
QW_DEV float4 cluster_load4(const float* p, int rank) {
    uint32_t addr;
    float4 v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

// Scratch: [0] tiles per share, [1 + b] first tile of sequence b; then the
// partials [2 shares][columns][D] and their (base exponent, sum); then the lse of a
// call that accumulates weights but returns none, and what the attention kernel keeps
// for the weights kernel (scores, or the tcgen05 form's Q operands).  (The tcgen05
// form has no plan.)
struct Scratch {
    int* plan;
    float* part;
    float2* ml;
    float* lse;
    float* kept;
    size_t bytes;
};
Scratch scratch_of(void* base, const Kv4View& c, int S, int Hq, size_t part_rows, size_t kept_bytes) {
    Scratch s;
    unsigned char* p = static_cast<unsigned char*>(base);
    auto take = [&](size_t n) {
        unsigned char* r = p;
        p += (n + 255) & ~(size_t)255;
        return r;
    };
    s.plan = reinterpret_cast<int*>(take((size_t)(c.batch + 1) * 4));
    s.part = reinterpret_cast<float*>(take(part_rows * c.D * 4));
    s.ml = reinterpret_cast<float2*>(take(part_rows * 8));
    s.lse = reinterpret_cast<float*>(take((size_t)c.batch * S * Hq * 4));
    s.kept = reinterpret_cast<float*>(take(kept_bytes));
    s.bytes = (size_t)(p - static_cast<unsigned char*>(base));
    return s;
}

QW_DEV int tiles_of(const Kv4Rows& r) { return (r.off + r.n + TK - 1) / TK; }

// How the call's tiles fall on the shares: sequence b's tiles are [first, first + heads * ncb * nt).
constexpr int WARP_SEQS = 128;  // up to here every warp works the plan out by itself

// A warp's view of up to WARP_SEQS sequences: lane l holds sequences 4 l .. 4 l + 3.
struct WarpPlan {
    int n[4], at, total;  // tiles of the lane's sequences, first tile of its first one, all tiles
    Kv4Rows rows[4];
    QW_DEV void make(const Kv4AttnArgs& a, int per_tile, bool report) {
        const int lane = threadIdx.x & 31;
        int s = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = 4 * lane + i;
            rows[i] = b < a.c.batch ? kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, a.err, report) : Kv4Rows{0, 0};
            n[i] = per_tile * tiles_of(rows[i]);
            s += n[i];
        }
        at = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += v;
        }
        total = __shfl_sync(0xffffffffu, at, 31);
        at -= s;
    }
    QW_DEV int first(int b) const {  // first tile of sequence b
        const int i = b & 3;
        int v = at + (i > 0 ? n[0] : 0) + (i > 1 ? n[1] : 0) + (i > 2 ? n[2] : 0);
        return __shfl_sync(0xffffffffu, v, b >> 2);
    }
};
QW_DEV int share_size(int total, int shares) { return max(1, (total + shares - 1) / shares); }

QW_DEV int block_sum(int v, int* red) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < AW; ++w) v += red[w];
    return v;
}
// Exclusive prefix over the block's threads.
QW_DEV int block_prefix(int v, int* red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 31) red[warp] = s;
    __syncthreads();
    s -= v;
    for (int w = 0; w < warp; ++w) s += red[w];
    return s;
}

struct Share {
    int begin, end;  // this block's tiles
    int b, b0;       // sequence of tile `begin` and its first tile
    Kv4Rows rw;      // its rows
};

// This block's share.  For many sequences block 0 leaves the plan to the joining kernel.
QW_DEV Share take_share(const Kv4AttnArgs& a, int ncb, int* plan) {
    const int B = a.c.batch, tid = threadIdx.x, per_tile = a.c.heads * ncb;
    Share s;
    if (B <= WARP_SEQS) {
        WarpPlan p;
        p.make(a, per_tile, blockIdx.x == 0 && tid < 32);
        const int per = share_size(p.total, gridDim.x);
        s.begin = min((long long)p.total, (long long)per * blockIdx.x);
        s.end = min(p.total, s.begin + per);
        s.b = B;
        s.b0 = 0;
        s.rw = {0, 0};
        int at = p.at;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned hit = __ballot_sync(0xffffffffu, at <= s.begin && s.begin < at + p.n[i]);
            if (hit) {
                const int l = __ffs(hit) - 1;
                s.b = 4 * l + i;
                s.b0 = __shfl_sync(0xffffffffu, at, l);
                s.rw.off = __shfl_sync(0xffffffffu, p.rows[i].off, l);
                s.rw.n = __shfl_sync(0xffffffffu, p.rows[i].n, l);
            }
            at += p.n[i];
        }
        return s;
    }
    __shared__ int red[AW], found[2];
    int total = 0;
    for (int b = tid; b < B; b += ANT)
        total += per_tile * tiles_of(kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, a.err, blockIdx.x == 0));
    total = block_sum(total, red);
    const int per = share_size(total, gridDim.x);
    s.begin = min((long long)total, (long long)per * blockIdx.x);
    s.end = min(total, s.begin + per);
    if (tid == 0) found[0] = B;
    if (blockIdx.x == 0 && tid == 0) plan[0] = per;
    int base = 0;
    for (int b0 = 0; b0 < B; b0 += ANT) {
        const int b = b0 + tid;
        const int n = b < B ? per_tile * tiles_of(kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, nullptr, false)) : 0;
        const int at = base + block_prefix(n, red);
        if (blockIdx.x == 0 && b < B) plan[1 + b] = at;
        if (at <= s.begin && s.begin < at + n) {
            found[0] = b;
            found[1] = at;
        }
        base += block_sum(n, red);
        if (blockIdx.x != 0 && base > s.begin) break;
    }
    __syncthreads();
    s.b = found[0];
    s.b0 = found[1];
    s.rw = s.b < B ? kv4_rows(a.seq_len, a.n_new, s.b, a.S, a.c.max_pos, nullptr, false) : Kv4Rows{0, 0};
    return s;
}

template <int D, int NT>
struct SplitSmem {
    static constexpr int CB = 8 * NT;
    static constexpr int RING = AW * ASTAGES * Tile<D>::BYTES;
    static constexpr int OLD = D + 4;  // output row of a warp's merge buffer, floats
    static constexpr int MERGE = AW * CB * OLD * 4, BLOCK = CB * (D * 4 + 8);  // + the block's own sums (cluster form)
    static constexpr int BYTES = (RING > MERGE + BLOCK ? RING : MERGE + BLOCK) + AW * CB * 8;
};

// The warp's columns of a column block (rows that a sequence turns out not to have are read and not used).
template <int D, int NT>
QW_DEV void fetch_cols(const Kv4AttnArgs& a, int b, int h, int cb, RawCol<D> (&raw)[NT]) {
    const int lane = threadIdx.x & 31, G = a.Hq / a.c.heads;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int c = cb * 8 * NT + 8 * n + (lane >> 2);
        fetch_col<D>(raw[n], c < G * a.S ? a.q + (b * a.qs.b + (c / G) * a.qs.s + (h * G + c % G) * a.qs.h) : nullptr, lane);
    }
}

// This warp's tiles first, first + step, ... below t1 of column block cb of (b, h):
// every warp has its own columns' state and its own ring of
// tiles (cp.async, so no warp waits for another).  Leaves (base exponent, sum) of every warp and column in
// wml and the warps' outputs, relative to the block's base, in wo.  WEIGHTS: the scores are kept too.
template <int D, int NT, bool WEIGHTS>
QW_DEV void run_tiles(const Kv4AttnArgs& a, const Kv4Rows& rw, int b, int h, int cb, const RawCol<D> (&raw)[NT], int first, int step, int t1,
                      unsigned char* smem, float* scores, int cp) {
    using L = Tile<D>;
    using SM = SplitSmem<D, NT>;
    constexpr int CB = SM::CB;
    float2* wml = reinterpret_cast<float2*>(smem + SM::BYTES - AW * CB * 8);  // [warp][column]
    float* wo = reinterpret_cast<float*>(smem);                               // [warp][column][OLD]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int G = a.Hq / a.c.heads, T = rw.off + rw.n;
    const uint32_t ring = smem_u32(smem) + warp * ASTAGES * L::BYTES;
    const unsigned char* ringp = smem + warp * ASTAGES * L::BYTES;
    const int mine = max(0, (t1 - first + step - 1) / step);
    TileLoader<D> loader;
    loader.start(head_rows<D>(a.c, (size_t)b * a.c.heads + h), first * TK, step, lane);
    const uint32_t lane_chunk = L::chunk_pos(lane / L::CPR, lane % L::CPR) * 16;
    int fill = 0;  // byte offset of the stage that the next tile goes to
    auto issue = [&](int k) {
        if (k < mine) loader.copy(ring + fill, ring + fill + lane_chunk, T, lane);
        cp_async_commit();
        fill = fill == (ASTAGES - 1) * L::BYTES ? 0 : fill + L::BYTES;
    };
#pragma unroll
    for (int k = 0; k < ASTAGES - 1; ++k) issue(k);

    Cols<D, NT> cols;
    State<D, NT> st;
    st.init();
    int vis[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        load_cols<D, NT>(cols, n, raw[n], a.scale, lane);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int ci = (cb * CB + 8 * n + 2 * t + e) / G;
            vis[n][e] = a.causal ? min(T, rw.off + ci + 1) : T;
        }
    }
    const int all = a.causal ? min(T, rw.off + cb * CB / G + 1) : T;  // keys that every column sees
    const unsigned char* tile = ringp;
    int key0 = first * TK;
    if (WEIGHTS) scores += (((size_t)b * a.c.heads + h) * a.c.max_pos + key0) * cp;
    for (int k = 0; k < mine; ++k) {
        cp_async_wait<ASTAGES - 2>();
        __syncwarp();
        issue(k + ASTAGES - 1);  // into the stage that the warp left in the turn before
        if (key0 + TK <= all)
            attend_tile<D, NT, false, WEIGHTS>(st, cols, tile, key0, T, vis, lane, scores, cp);
        else
            attend_tile<D, NT, true, WEIGHTS>(st, cols, tile, key0, T, vis, lane, scores, cp);
        key0 += step * TK;
        if (WEIGHTS) scores += (size_t)(step * TK) * cp;
        tile = tile == ringp + (ASTAGES - 1) * L::BYTES ? ringp : tile + L::BYTES;
        __syncwarp();
    }
    cp_async_wait<0>();
    if (mine > 0) reduce_lanes(st);
    if (g == 0)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) wml[warp * CB + 8 * n + 2 * t + e].x = st.base(n, e);
    __syncthreads();  // also: every warp has left its ring
    if (mine > 0)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int col = 8 * n + 2 * t + e;
                float M = wml[col].x;
#pragma unroll
                for (int w = 1; w < AW; ++w) M = fmaxf(M, wml[w * CB + col].x);
                const float f = half_pow(st.base(n, e) - M);
                if (g == 0) wml[warp * CB + col].y = st.l[n][e] * f * f;
                float* dst = wo + (warp * CB + col) * SM::OLD + 4 * g;
#pragma unroll
                for (int gr = 0; gr < D / 64; ++gr)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 v = out_pair(st, gr, i, n, e);
                        *reinterpret_cast<float2*>(dst + 64 * gr + 32 * (i >> 1) + 2 * (i & 1)) = make_float2(v.x * f * f, v.y * f * f);
                    }
            }
    __syncthreads();
}

// Sum over the block's first `warps` warps (those that had tiles) of column col, dimensions d .. d + 3,
// relative to the block's base M.
template <int D, int NT>
QW_DEV float4 warps_sum(const unsigned char* smem, int warps, int col, int d, float& M, float& l) {
    using SM = SplitSmem<D, NT>;
    const float2* wml = reinterpret_cast<const float2*>(smem + SM::BYTES - AW * SM::CB * 8);
    const float* wo = reinterpret_cast<const float*>(smem);
    M = M0;
    l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w0 = 0; w0 < AW; w0 += 4) {
        float2 ml[4];
        float4 v[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            ml[w] = w0 + w < warps ? wml[(w0 + w) * SM::CB + col] : make_float2(M0, 0.f);
            v[w] = w0 + w < warps ? *reinterpret_cast<const float4*>(wo + ((w0 + w) * SM::CB + col) * SM::OLD + d)
                                  : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            M = fmaxf(M, ml[w].x);
            l += ml[w].y;
            o.x += v[w].x;
            o.y += v[w].y;
            o.z += v[w].z;
            o.w += v[w].w;
        }
    }
    return o;
}

// Output of column c, dimensions d .. d + 3, from its sums.
QW_DEV void write_out(const Kv4AttnArgs& a, const Kv4Rows& rw, int b, int h, int c, int d, float4 o, float M, float l) {
    const int G = a.Hq / a.c.heads, i = c / G;
    const bool has = i < rw.n && l != 0.f;
    const float inv = has ? 1.f / l : 0.f;
    bf16* dst = a.out + (b * a.os.b + i * a.os.s + (h * G + c % G) * a.os.h) + d;
    *reinterpret_cast<uint2*>(dst) = has ? make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv)) : make_uint2(0u, 0u);
    if (d == 0 && a.lse) a.lse[((size_t)b * a.S + i) * a.Hq + h * G + c % G] = has ? (M + log2f(l)) * LN2 : -INFINITY;
}

// 131071 keys, 8 kv heads, 4 columns each: 34.4 us of the call's 37.4 = 4.4 TB/s (the keys themselves at 5.8 TB/s; ~10 us are the
// plan, the queries, the ring's start and the merges); the issue slots are 59 % taken, half of that by unpacking
// nibbles.  A warp of its own for every tile, with no barrier on the way, because 16 warps in step took 39.6 us.
template <int D, int NT, bool WEIGHTS>
__global__ void __launch_bounds__(ANT, NT == 1 ? 2 : 1) kv4_attn_split_kernel(const Kv4AttnArgs a, int ncb, int* plan, float* part, float2* pml,
                                                                              float* scores, int cp) {
    constexpr int CB = 8 * NT;
    extern __shared__ __align__(128) unsigned char smem[];
    const int tid = threadIdx.x, C = a.Hq / a.c.heads * a.S;
    pdl_wait();
    // the dependent kernel's blocks may settle in: they wait for this kernel's end before they touch what it
    // writes, and read the lengths and the cache, which only earlier kernels write, while it runs
    pdl_launch_dependents();
    const Share sh = take_share(a, ncb, plan);
    int u = sh.begin, b0 = sh.b0, b = sh.b;
    Kv4Rows rw = sh.rw;
    while (u < sh.end) {
        const int nt = tiles_of(rw);
        const int nseq = nt * a.c.heads * ncb;
        if (u >= b0 + nseq) {  // the next sequence (some are empty)
            b0 += nseq;
            ++b;
            rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, nullptr, false);
            continue;
        }
        const int seg = (u - b0) / nt, t0 = u - b0 - seg * nt;
        const int t1 = min(nt, t0 + (sh.end - u));
        const int h = ncb == 1 ? seg : seg / ncb, cb = seg - h * ncb;
        RawCol<D> raw[NT];
        fetch_cols<D, NT>(a, b, h, cb, raw);
        run_tiles<D, NT, WEIGHTS>(a, rw, b, h, cb, raw, t0 + (tid >> 5), AW, t1, smem, scores, cp);
        const bool whole = t0 == 0 && t1 == nt;
        const size_t slot = 2 * (size_t)blockIdx.x + (u == sh.begin ? 0 : 1);
        for (int idx = tid; idx < CB * (D / 4); idx += ANT) {
            const int col = idx / (D / 4), d = 4 * (idx % (D / 4)), c = cb * CB + col;
            if (c >= C) break;
            float M, l;
            const float4 o = warps_sum<D, NT>(smem, min(AW, t1 - t0), col, d, M, l);
            if (whole) {
                write_out(a, rw, b, h, c, d, o, M, l);
            } else {
                *reinterpret_cast<float4*>(part + (slot * CB + col) * D + d) = o;
                if (d == 0) pml[slot * CB + col] = make_float2(M, l);
            }
        }
        __syncthreads();  // the merge buffer is the ring
        u += t1 - t0;
    }
}

// Short caches: a cluster of `cluster` blocks takes a whole segment, tile k by block k % cluster, and joins
// through distributed shared memory -- one launch and no partials in memory.  32 sequences of up to 2048 keys, 2 kv
// heads: 7.5 us; 5 rows of 32 heads on 812 keys: 8.6 us.
template <int D, int NT, bool WEIGHTS>
__global__ void __launch_bounds__(ANT, NT == 1 ? 2 : 1) kv4_attn_cluster_kernel(const Kv4AttnArgs a, int ncb, int cluster, float* scores, int cp) {
    using SM = SplitSmem<D, NT>;
    constexpr int CB = SM::CB;
    extern __shared__ __align__(128) unsigned char smem[];
    float* bo = reinterpret_cast<float*>(smem + SM::MERGE);       // [column][D] of this block
    float2* bml = reinterpret_cast<float2*>(bo + CB * D);         // [column]
    pdl_wait();
    pdl_launch_dependents();
    const int tid = threadIdx.x, C = a.Hq / a.c.heads * a.S;
    const int rank = blockIdx.x % cluster, seg = blockIdx.x / cluster;
    const int cb = seg % ncb, h = seg / ncb % a.c.heads, b = seg / ncb / a.c.heads;
    RawCol<D> raw[NT];
    fetch_cols<D, NT>(a, b, h, cb, raw);  // before the length arrives
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, a.err, rank == 0 && h == 0 && cb == 0 && tid == 0);
    run_tiles<D, NT, WEIGHTS>(a, rw, b, h, cb, raw, (tid >> 5) * cluster + rank, AW * cluster, tiles_of(rw), smem, scores, cp);
    const int nt = tiles_of(rw);
    for (int idx = tid; idx < CB * (D / 4); idx += ANT) {
        const int col = idx / (D / 4), d = 4 * (idx % (D / 4)), c = cb * CB + col;
        if (c >= C) break;
        float M, l;  // warp w has tiles when w * cluster + rank < nt
        const float4 o = warps_sum<D, NT>(smem, max(0, min(AW, (nt - rank + cluster - 1) / cluster)), col, d, M, l);
        if (cluster == 1) {
            write_out(a, rw, b, h, c, d, o, M, l);
        } else {
            *reinterpret_cast<float4*>(bo + col * D + d) = o;
            if (d == 0) bml[col] = make_float2(M, l);
        }
    }
    if (cluster == 1) return;
    cluster_sync();
    for (int idx = rank * ANT + tid; idx < CB * (D / 4); idx += cluster * ANT) {
        const int col = idx / (D / 4), d = 4 * (idx % (D / 4)), c = cb * CB + col;
        if (c >= C) break;
        float2 ml[MAX_CLUSTER];
        float4 v[MAX_CLUSTER];
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; ++r) {
            ml[r] = r < cluster ? cluster_load2(&bml[col].x, r) : make_float2(M0, 0.f);
            v[r] = r < cluster ? cluster_load4(&bo[col * D + d], r) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float M = M0, l = 0.f;
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; ++r) M = fmaxf(M, ml[r].x);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int r = 0; r < MAX_CLUSTER; ++r) {
            const float f = half_pow(ml[r].x - M);
            l = fmaf(ml[r].y * f, f, l);
            o.x = fmaf(v[r].x * f, f, o.x);
            o.y = fmaf(v[r].y * f, f, o.y);
            o.z = fmaf(v[r].z * f, f, o.z);
            o.w = fmaf(v[r].w * f, f, o.w);
        }
        write_out(a, rw, b, h, c, d, o, M, l);
    }
    cluster_sync();  // the blocks' sums are read until here
}

// Joins the partials of segments that span shares, and writes the rows of empty
// sequences.  One block per (column, sequence); every warp works out the
// segment's shares by itself.
constexpr int JOIN_WARPS = 8;
template <int D>
__global__ void __launch_bounds__(32 * JOIN_WARPS) kv4_attn_join_kernel(const Kv4AttnArgs a, int cb_size, int ncb, int shares, const int* plan,
                                                                        const float* part, const float2* pml) {
    __shared__ float sh[JOIN_WARPS * (D + 2)];
    const int b = blockIdx.y, G = a.Hq / a.c.heads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int h = blockIdx.x % a.Hq, i = blockIdx.x / a.Hq;  // query head, row
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, nullptr, false);
    const int nt = tiles_of(rw);
    int per, s0;
    if (a.c.batch <= WARP_SEQS) {  // before the wait: the lengths are not this call's
        WarpPlan p;
        p.make(a, a.c.heads * ncb, false);
        per = share_size(p.total, shares);
        s0 = p.first(b);
        pdl_wait();
    } else {
        pdl_wait();
        per = plan[0];
        s0 = plan[1 + b];
    }
    bf16* dst = a.out + (b * a.os.b + i * a.os.s + h * a.os.h);
    float* lse = a.lse ? a.lse + ((size_t)b * a.S + i) * a.Hq + h : nullptr;
    if (nt == 0 || i >= rw.n) {
        if (warp == 0 && lane < D / 8) *reinterpret_cast<uint4*>(dst + 8 * lane) = make_uint4(0u, 0u, 0u, 0u);
        if (lse && threadIdx.x == 0) *lse = -INFINITY;
        return;
    }
    const int c = i * G + h % G, cb = c / cb_size, col = c % cb_size;
    s0 += ((h / G) * ncb + cb) * nt;
    const int first = s0 / per, last = (s0 + nt - 1) / per;
    if (first == last) return;
    // the first share's partial of this segment is its second one if the share began before it
    auto slot = [&](int k) { return (2ll * (first + k) + (k == 0 && first * per < s0 ? 1 : 0)) * cb_size + col; };
    join_row<D, JOIN_WARPS, 8>(last - first + 1, warp, slot, part, pml, sh, dst, lse);
}

// ---- attention weights ------------------------------------------------------
// A key's weight is summed by one lane quad in a fixed order, over the scores recomputed from the K rows and
// the rows' log-sum-exp.

// K rows of keys key0 + 8 r + g (r < 2 KB) straight from memory, in the layout of read_keys; zeros from T on.
template <int D, int KB>
struct MassKeys {
    KeyBlock<D> w[KB];
    uint32_t s[2 * KB], z[2 * KB];
};
template <int D, int KB>
QW_DEV void fetch_keys(MassKeys<D, KB>& o, const Kv4View& c, size_t bh, int key0, int T, int lane) {
    constexpr int GR = D / 64;
    const int g = lane >> 2, t = lane & 3;
    const uint32_t* w = c.p[0].w + bh * c.max_pos * (D / 8);
    const unsigned char* s = reinterpret_cast<const unsigned char*>(c.p[0].s) + bh * c.max_pos * (2 * GR);
    const unsigned char* z = reinterpret_cast<const unsigned char*>(c.p[0].b) + bh * c.max_pos * (2 * GR);
#pragma unroll
    for (int r = 0; r < 2 * KB; ++r) {
        const int k = key0 + 8 * r + g;
        const bool ok = k < T;
#pragma unroll
        for (int gr = 0; gr < GR; ++gr)
#pragma unroll
            for (int j = 0; j < 2; ++j) o.w[r >> 1].w[gr][r & 1][j] = ok ? w[(size_t)k * (D / 8) + 8 * gr + 4 * j + t] : 0u;
        const size_t at = (size_t)k * (2 * GR);
        o.s[r] = !ok ? 0u : GR == 2 ? *reinterpret_cast<const uint32_t*>(s + at) : (uint32_t)*reinterpret_cast<const uint16_t*>(s + at);
        o.z[r] = !ok ? 0u : GR == 2 ? *reinterpret_cast<const uint32_t*>(z + at) : (uint32_t)*reinterpret_cast<const uint16_t*>(z + at);
    }
}
// Adds the probabilities of the keys in the columns of n-tile n to sum[r]; base = -log2 of the rows' sums
// (-inf: no column), vis the keys a column sees.
template <int D, int KB, int NT>
QW_DEV void add_weights(float (&sum)[2 * KB], const MassKeys<D, KB>& k, const Cols<D, NT>& cols, const float (&base)[NT][4],
                        const int (&vis)[NT][2], int key0, int lane) {
    constexpr int GR = D / 64;
    const int g = lane >> 2;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
        float acc[GR][NT][4];
        key_dots<D, NT>(acc, k.w[kb], cols);
        float ks[2][GR];
        unpack<GR>(k.s[2 * kb], ks[0]);
        unpack<GR>(k.s[2 * kb + 1], ks[1]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float x[4];
            mma_bf16_k8(x, k.z[2 * kb], k.z[2 * kb + 1], cols.qb[n], base[n]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float d = ks[e >> 1][0] * acc[0][n][e];
                if (GR == 2) d = fmaf(ks[e >> 1][GR - 1], acc[GR - 1][n][e], d);
                const float p = ex2(fmaf(cols.c[n][e & 1], d, x[e]));
                const int r = 2 * kb + (e >> 1);
                sum[r] += key0 + 8 * r + g < vis[n][e & 1] ? p : 0.f;
            }
        }
    }
}
// Sum over the lane quad of a key; lane t of the quad adds row r = t to mass.
template <int KB>
QW_DEV void store_weights(float (&sum)[2 * KB], float* mass, int key0, int T, int lane) {
    static_assert(2 * KB <= 4, "a lane of the quad for every row");
#pragma unroll
    for (int r = 0; r < 2 * KB; ++r) {
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 1);
        sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], 2);
    }
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int r = 0; r < 2 * KB; ++r)
        if (t == r && key0 + 8 * r + g < T) mass[key0 + 8 * r + g] += sum[r];
}

// Up to SCORE_COLUMNS columns: the attention kernels leave their scores [batch][kv head][key][cp] (base 2; at eight
// columns 32 bytes a key next to the 72 of its K row), so that this pass reads them from L2 and takes no products.
// 4 sequences of up to 16000 keys, 8 columns: 28.9 us with the attention, 39.0 us with scores recomputed from K.
// A thread adds one key's columns in their order.
constexpr int SCORE_COLUMNS = 16, WNT = 256;
template <int VEC>
__global__ void __launch_bounds__(WNT) kv4_mass_scores_kernel(const Kv4AttnArgs a, const float* scores, int cp) {
    __shared__ float base[SCORE_COLUMNS];  // the columns' log2-sum-exp
    __shared__ int seen[SCORE_COLUMNS];    // the keys that they see (a NaN row's others have no weight from it); 0 for padding
    const int h = blockIdx.y, b = blockIdx.z, G = a.Hq / a.c.heads, C = G * a.S, key = blockIdx.x * WNT + threadIdx.x;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, nullptr, false);
    const int T = rw.off + rw.n;
    pdl_wait();
    if (blockIdx.x * WNT >= T) return;
    if (threadIdx.x < cp) {
        const int c = threadIdx.x, i = c / G;
        const bool row = c < C && i < rw.n;
        base[c] = row ? a.lse[((size_t)b * a.S + i) * a.Hq + h * G + c % G] * LOG2E : 0.f;
        seen[c] = !row ? 0 : a.causal ? min(T, rw.off + i + 1) : T;
    }
    const size_t at = ((size_t)b * a.c.heads + h) * a.c.max_pos + key;
    const bool ok = key < T;
    float v[SCORE_COLUMNS];
    const float before = ok ? a.mass[at] : 0.f;
#pragma unroll
    for (int c = 0; c < SCORE_COLUMNS; c += VEC)
        if (ok && c < cp) {
            if (VEC == 4)
                *reinterpret_cast<float4*>(v + c) = *reinterpret_cast<const float4*>(scores + at * cp + c);
            else
                *reinterpret_cast<float2*>(v + c) = *reinterpret_cast<const float2*>(scores + at * cp + c);
        }
    __syncthreads();
    if (!ok) return;
    float sum = 0.f;
#pragma unroll
    for (int c = 0; c < SCORE_COLUMNS; ++c)
        if (c < cp) sum += key < seen[c] ? ex2(v[c] - base[c]) : 0.f;
    a.mass[at] = before + sum;
}

// 17 to 63 columns: a warp keeps 16 keys (eight warps of 16: with 32 a chunk of 512 rows on 4096 keys left half of the
// GPU without a second block per SM) and the block walks the columns, 64 at a time, one n-tile prepared by each warp
// while the queries of the next 64 are in flight.
constexpr int MC = 8;
template <int D>
__global__ void __launch_bounds__(ANT, 2) kv4_mass_kernel(const Kv4AttnArgs a) {
    constexpr int GR = D / 64, MK = 16;
    __shared__ uint32_t sf[MC][GR * 4 * 2][32];  // n-tile, fragment register, lane
    __shared__ float sc[MC][3][8];               // n-tile, {c, -log2 of the sum, keys seen}, column
    __shared__ uint32_t sq[MC][32];              // n-tile, bias operand, lane
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y, b = blockIdx.z, G = a.Hq / a.c.heads;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, nullptr, false);
    const int T = rw.off + rw.n;
    const int block0 = blockIdx.x * AW * MK, key0 = block0 + warp * MK;
    if (block0 >= T) {
        pdl_wait();
        return;
    }
    const size_t bh = (size_t)b * a.c.heads + h;
    MassKeys<D, 1> keys;
    fetch_keys<D, 1>(keys, a.c, bh, key0, T, lane);
    float sum[2] = {0.f, 0.f};
    // columns that see none of the block's keys come first when causal: skip them
    const int c_first = a.causal ? max(0, block0 - rw.off) * G / 8 * 8 : 0, c_end = rw.n * G;
    RawCol<D> raw;
    auto fetch = [&](int c0) {
        const int c = c0 + 8 * warp + g;
        fetch_col<D>(raw, c < c_end ? a.q + (b * a.qs.b + (c / G) * a.qs.s + (h * G + c % G) * a.qs.h) : nullptr, lane);
    };
    fetch(c_first);
    pdl_wait();  // the rows' log-sum-exp are the attention kernel's
    for (int c0 = c_first; c0 < c_end; c0 += 8 * MC) {
        const int cw = c0 + 8 * warp + g, iw = cw / G;
        const float lse = t == 0 && cw < c_end ? a.lse[((size_t)b * a.S + iw) * a.Hq + h * G + cw % G] : INFINITY;
        Cols<D, 1> o;
        load_cols<D, 1>(o, 0, raw, a.scale, lane);
        fetch(c0 + 8 * MC);
        __syncthreads();
#pragma unroll
        for (int gr = 0; gr < GR; ++gr)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sf[warp][(gr * 4 + j) * 2][lane] = o.f[gr][j][0][0];
                sf[warp][(gr * 4 + j) * 2 + 1][lane] = o.f[gr][j][0][1];
            }
        if (g == 0)
#pragma unroll
            for (int e = 0; e < 2; ++e) sc[warp][0][2 * t + e] = o.c[0][e];
        sq[warp][lane] = o.qb[0];
        if (t == 0) {
            sc[warp][1][g] = -lse * LOG2E;
            sc[warp][2][g] = __int_as_float(cw < c_end ? (a.causal ? min(T, rw.off + iw + 1) : T) : 0);
        }
        __syncthreads();
        if (key0 >= T) continue;
        const int nn = min(MC, (c_end - c0 + 7) / 8);
        for (int n = 0; n < nn; ++n) {
            Cols<D, 1> cols;
            float base[1][4];
            int vis[1][2];
            cols.qb[0] = sq[n][lane];
#pragma unroll
            for (int gr = 0; gr < GR; ++gr)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    cols.f[gr][j][0][0] = sf[n][(gr * 4 + j) * 2][lane];
                    cols.f[gr][j][0][1] = sf[n][(gr * 4 + j) * 2 + 1][lane];
                }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                cols.c[0][e] = sc[n][0][2 * t + e];
                base[0][e] = base[0][2 + e] = sc[n][1][2 * t + e];
                vis[0][e] = __float_as_int(sc[n][2][2 * t + e]);
            }
            add_weights<D, 1, 1>(sum, keys, cols, base, vis, key0, lane);
        }
    }
    store_weights<1>(sum, a.mass + bh * a.c.max_pos, key0, T, lane);
}

// Form of a call: from TC_COLUMNS columns per kv head the tcgen05 kernel, below it the split kernel
// with column blocks of 8 (two blocks of threads per SM) or 16.  32768 keys, 8 kv heads: 43.0 us at 48 columns, 53.9 at 60
// (four column blocks unpack the keys four times), 52.5 at 64 and 52.8 at 128 by the tcgen05 kernel.
constexpr int TC_COLUMNS = 64;
constexpr int CLUSTER_TILES = 4;
struct Shape {
    bool tc;
    TcShape t;
    int nt, cb, ncb, shares;
    int cp;       // columns of a kept score row, 0: the scores are not kept
    size_t kept_bytes;
    int cluster;  // blocks of a segment in the cluster form, 0: shares
    size_t part_rows;
};
Shape shape_of(const Kv4View& c, int S, int Hq, int num_sms) {
    const long long C = (long long)(Hq / c.heads) * S;
    Shape s = {};
    s.tc = C >= TC_COLUMNS;
    if (s.tc) {
        s.t = kv4_tc_shape(c, S, Hq, num_sms);
        s.part_rows = s.t.part_rows;
        s.kept_bytes = s.t.kept_bytes;
        return s;
    }
    s.nt = C <= 8 ? 1 : 2;
    s.cb = 8 * s.nt;
    s.ncb = (int)((C + s.cb - 1) / s.cb);
    s.cp = C <= SCORE_COLUMNS ? (int)(C + 1) / 2 * 2 : 0;
    s.kept_bytes = (size_t)c.batch * c.heads * c.max_pos * s.cp * 4;
    s.shares = s.nt == 1 ? 2 * num_sms : num_sms;
    // The cluster form, when the longest sequence the cache can hold is at most CLUSTER_TILES tiles a warp (what a
    // ragged batch loses to its longest sequence then costs less than the joining kernel) and its blocks fit at once.
    const long long segs = (long long)c.batch * c.heads * s.ncb;
    const int most = (c.max_pos + TK - 1) / TK;
    int cl = 1;
    // (clusters of 8 are counted on three quarters of the SMs: what is left of a GPC holds none; 5 rows on 812 keys
    // with clusters that did not fit at once: 1.6 times as long)
    while (cl < MAX_CLUSTER && segs * 2 * cl * (cl == 4 ? 4 : 3) <= 3ll * s.shares && most > AW * cl) cl *= 2;
    if (most <= CLUSTER_TILES * AW * cl && segs * cl <= 0x7FFFFFFF) {
        s.cluster = cl;
        return s;
    }
    s.part_rows = (size_t)2 * s.shares * s.cb;
    return s;
}

template <int D, int NT, bool WEIGHTS>
cudaError_t launch_split(const Kv4AttnArgs& a, const Shape& sp, const Scratch& sc, cudaStream_t st) {
    constexpr int smem = SplitSmem<D, NT>::BYTES;
    if (sp.cluster) {
        const cudaError_t e = ensure_max_dyn_smem(kv4_attn_cluster_kernel<D, NT, WEIGHTS>, smem);
        if (e != cudaSuccess) return e;
        const unsigned blocks = (unsigned)(sp.cluster * sp.ncb * a.c.heads) * (unsigned)a.c.batch;
        return launch(kv4_attn_cluster_kernel<D, NT, WEIGHTS>, dim3(blocks), dim3(ANT), smem, sp.cluster, st, a, sp.ncb, sp.cluster, sc.kept,
                      sp.cp);
    }
    cudaError_t e = ensure_max_dyn_smem(kv4_attn_split_kernel<D, NT, WEIGHTS>, smem);
    if (e != cudaSuccess) return e;
    e = launch(kv4_attn_split_kernel<D, NT, WEIGHTS>, dim3(sp.shares), dim3(ANT), smem, 1, st, a, sp.ncb, sc.plan, sc.part, sc.ml, sc.kept,
               sp.cp);
    if (e != cudaSuccess) return e;
    return launch(kv4_attn_join_kernel<D>, dim3((unsigned)(a.S * a.Hq), a.c.batch), dim3(32 * JOIN_WARPS), 0, 1, st, a, sp.cb, sp.ncb,
                  sp.shares, (const int*)sc.plan, (const float*)sc.part, (const float2*)sc.ml);
}

template <int D>
cudaError_t launch_d(const Kv4AttnArgs& a, const Shape& sp, const Scratch& sc, cudaStream_t st) {
    if (sp.tc) return launch_kv4_attn_tc(a, sp.t, sc.part, sc.ml, sc.kept, st);
    const bool keep = a.mass && sp.cp;
    const cudaError_t e = sp.nt == 1 ? (keep ? launch_split<D, 1, true>(a, sp, sc, st) : launch_split<D, 1, false>(a, sp, sc, st))
                                     : (keep ? launch_split<D, 2, true>(a, sp, sc, st) : launch_split<D, 2, false>(a, sp, sc, st));
    if (e != cudaSuccess || !a.mass) return e;
    if (keep) {
        const dim3 grid((a.c.max_pos + WNT - 1) / WNT, a.c.heads, a.c.batch);
        return launch(sp.cp % 4 == 0 ? kv4_mass_scores_kernel<4> : kv4_mass_scores_kernel<2>, grid, dim3(WNT), 0, 1, st, a,
                      (const float*)sc.kept, sp.cp);
    }
    const dim3 grid((a.c.max_pos + AW * 16 - 1) / (AW * 16), a.c.heads, a.c.batch);
    return launch(kv4_mass_kernel<D>, grid, dim3(ANT), 0, 1, st, a);
}

}  // namespace

size_t kv4_attn_scratch_bytes(const Kv4View& c, int S, int Hq, int num_sms) {
    const Shape sp = shape_of(c, S, Hq, num_sms);
    return scratch_of(nullptr, c, S, Hq, sp.part_rows, sp.kept_bytes).bytes;
}

cudaError_t launch_kv4_attention(const Kv4AttnArgs& in, void* scratch, int num_sms, cudaStream_t st) {
    Kv4AttnArgs a = in;
    const Shape sp = shape_of(a.c, a.S, a.Hq, num_sms);
    // tiles are counted in 32 bits (180 GB of cache are less than 2^26 tiles of one column block)
    if (!sp.tc && !sp.cluster && (long long)a.c.batch * a.c.heads * sp.ncb * ((a.c.max_pos + TK - 1) / TK) > 0x7FFFFFFF) return cudaErrorInvalidValue;
    const Scratch sc = scratch_of(scratch, a.c, a.S, a.Hq, sp.part_rows, sp.kept_bytes);
    if (a.mass && !a.lse) a.lse = sc.lse;
    return a.c.D == 128 ? launch_d<128>(a, sp, sc, st) : launch_d<64>(a, sp, sc, st);
}

}  // namespace qw
