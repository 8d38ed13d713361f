// Eviction from the 4-bit KV cache by accumulated attention weight.
//
// Per (sequence, kv head) of length n > keep: the last `recent` positions stay,
// and of the others the keep - recent with the largest weight (the lower
// position wins a tie).  The kept rows move to the front in position order,
// with their weights; n <= keep keeps every row.
//
//   1. select: weights become unsigned keys of the same order.  A thread block
//      holds the keys of a (sequence, head) in shared memory, 16384 of them; more
//      positions take a cluster of blocks, a slice each.  Three histogram passes
//      (11, 11 and 10 bits, summed over the cluster through distributed shared
//      memory) find the threshold key and how many of its equals stay; votes rank
//      the kept positions.
//   2. move: dst row r = src row index[r].
//
// 8 sequences of up to 16384 positions, 8 heads, half of them kept: 41 us, of them
// 24 for the move (117 MB at 4.8 TB/s, waiting on its gathers) and 14 for the
// selection, which is bound by the latency of its passes (with clusters of four
// blocks 16: a cluster barrier and the remote reads behind it take 1.8 us).
#include <algorithm>

#include "kv4.h"
#include "kv4_launch.h"
#include "smem_attr.h"

namespace qw {
namespace {

constexpr int SEL_NT = 1024, SEL_W = SEL_NT / 32;
constexpr int BINS = 2048;
constexpr int SEL_MAX_CLUSTER = 8;
constexpr int SLICE = 16384;             // keys a block holds in shared memory; further ones are read again per pass

// Unsigned key of the same order as the float; -0 equals +0, NaN is above everything.
QW_DEV uint32_t order_key(float v) {
    uint32_t u = __float_as_uint(v);
    if (v != v) return 0xFFFFFFFFu;
    if ((u << 1) == 0u) u = 0u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// A length out of range counts as an empty sequence, as in kv4_rows.
QW_DEV int length_of(const Kv4EvictArgs& a, int b) {
    const int n = a.seq_len[b];
    return n < 0 || n > a.src.max_pos ? 0 : n;
}

QW_DEV void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
// Ints at `p` in the cluster's block `rank`.
QW_DEV uint32_t cluster_addr(const int* p, int rank) {
    uint32_t addr;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(p)), "r"(rank));
    return addr;
}
QW_DEV int2 cluster_load2(const int* p, int rank) {
    int2 v;
    asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(cluster_addr(p, rank)) : "memory");
    return v;
}
// index[b][h][0..new length): the kept positions in increasing order.
__global__ void __launch_bounds__(SEL_NT, 1) kv4_select_kernel(const Kv4EvictArgs a, int cluster, int* index, int* count) {
    extern __shared__ __align__(16) int sel_smem[];
    int* hist = sel_smem;                                             // [3][BINS]
    uint32_t* held = reinterpret_cast<uint32_t*>(sel_smem + 3 * BINS);  // keys of the slice's first SLICE positions
    __shared__ int2 red[32], tally;
    __shared__ int wsum[3][32], pick[3][2];
    const int rank = blockIdx.x % cluster, h = blockIdx.x / cluster, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31,
              warp = tid >> 5;
    pdl_wait();
    pdl_launch_dependents();
    const int n = length_of(a, b);
    const size_t bh = (size_t)b * a.src.heads + h;
    int* idx = index + bh * a.keep;
    int* out = a.index_out ? a.index_out + bh * a.keep : nullptr;
    if (tid == 0 && h == 0 && rank == 0) count[b] = min(n, a.keep);
    if (n <= a.keep) {  // the whole cluster takes this branch
        for (int r = rank * SEL_NT + tid; r < a.keep; r += cluster * SEL_NT) {
            const int v = r < n ? r : -1;
            idx[r] = v;
            if (out) out[r] = v;
        }
        return;
    }
    // as many blocks of the cluster as the positions need (each cluster barrier costs a microsecond)
    const int active = min(cluster, (n + SLICE - 1) / SLICE);
    if (active == 1 && rank > 0) return;
    const float* mass = a.mass_src + bh * a.src.max_pos;
    const int old = n - a.recent, want = a.keep - a.recent;
    const int slice = (n + active - 1) / active, j0 = min(n, rank * slice), j1 = min(n, j0 + slice);
    const int jo = max(j0, min(j1, old));  // [j0, jo): may be dropped; [jo, j1): recent
    // A warp takes consecutive positions [w0, w1), a lane every 32nd of them.
    const int span = ((slice + SEL_W - 1) / SEL_W + 31) & ~31, w0 = min(j1, j0 + warp * span), w1 = min(j1, w0 + span);
    auto load = [&](int j) { return j < w1 && j < jo ? mass[j] : 0.f; };
    const int most = min(w1, j0 + SLICE);  // [w0, most): held
    for (int j = w0 + lane; j < most; j += 32 * 8) {  // eight loads in flight
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = load(j + 32 * e);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (j + 32 * e < most) held[j + 32 * e - j0] = order_key(v[e]);
    }
    for (int i = tid; i < 3 * BINS / 4; i += SEL_NT) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    // f(position, key) of the warp's positions, by whole warps.  (Rolled, as the passes are: the block is short and
    // runs at the pace of instruction fetch; with 16 keys a thread in registers it took 12.3 us for 700 positions.)
    auto each = [&](auto f) {
        int j = w0;
#pragma unroll 1
        for (; j + 128 <= most; j += 128) {
            uint32_t k[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) k[e] = held[j + 32 * e + lane - j0];
#pragma unroll
            for (int e = 0; e < 4; ++e) f(j + 32 * e + lane, k[e]);
        }
#pragma unroll 1
        for (; j < w1; j += 32) f(j + lane, j + lane < most ? held[j + lane - j0] : order_key(load(j + lane)));
    };
    uint32_t prefix = 0;
    int left = want;
    if (want > 0) {
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
            const uint32_t mask = pass == 2 ? 1023u : 2047u;
            const int above_bits = pass == 0 ? 31 : pass == 1 ? 21 : 10;  // every higher digit has to agree
            int* hp = hist + pass * BINS;
            each([&](int j, uint32_t k) {
                if (j < w1 && j < jo && (pass == 0 || (k >> above_bits) == (prefix >> above_bits))) atomicAdd(&hp[(k >> shift) & mask], 1);
            });
            if (active > 1)
                cluster_sync();
            else
                __syncthreads();
            // warp w counts the 64 bins from 64 (31 - w) on, lane l two of them from 2 (31 - l) on: warps, lanes
            // and c[0], c[1] in order from the largest digit down
            static_assert(BINS == 2 * SEL_NT, "two bins per thread");
            const int d0 = 64 * (SEL_W - 1 - warp) + 2 * (31 - lane);
            int c[2] = {0, 0};
            if (active > 1) {
                int2 v[SEL_MAX_CLUSTER];
#pragma unroll
                for (int r = 0; r < SEL_MAX_CLUSTER; ++r) v[r] = r < active ? cluster_load2(&hp[d0], r) : make_int2(0, 0);
#pragma unroll
                for (int r = 0; r < SEL_MAX_CLUSTER; ++r) {
                    c[0] += v[r].y;
                    c[1] += v[r].x;
                }
            } else {
                const int2 v = *reinterpret_cast<const int2*>(&hp[d0]);
                c[0] = v.y, c[1] = v.x;
            }
            const int own = c[0] + c[1], mine = __reduce_add_sync(0xffffffffu, own);
            if (lane == 0) wsum[pass][warp] = mine;
            __syncthreads();
            const int before = __reduce_add_sync(0xffffffffu, lane < warp ? wsum[pass][lane] : 0);
            if (before < left && left <= before + mine) {  // this warp's bins hold the threshold
                int s = own;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, s, o);
                    if (lane >= o) s += v;
                }
                int above = before + s - own;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (above < left && left <= above + c[e]) {
                        pick[pass][0] = d0 + 1 - e;
                        pick[pass][1] = left - above;
                    }
                    above += c[e];
                }
            }
            __syncthreads();
            prefix |= (uint32_t)pick[pass][0] << shift;
            left = pick[pass][1];
        }
    }
    // The kept positions ranked by votes: positions that stay for certain, and those that equal the threshold.
    const unsigned below = (1u << lane) - 1u;
    auto votes = [&](int j, uint32_t k, unsigned& above, unsigned& equal) {
        const bool in = j < w1, low = in && j < jo && want > 0;
        above = __ballot_sync(0xffffffffu, (in && j >= jo) || (low && k > prefix));
        equal = __ballot_sync(0xffffffffu, low && k == prefix);
    };
    int2 mine = make_int2(0, 0);
    each([&](int j, uint32_t k) {
        unsigned above, equal;
        votes(j, k, above, equal);
        mine.x += __popc(above);
        mine.y += __popc(equal);
    });
    if (lane == 0) red[warp] = mine;
    __syncthreads();
    const int2 p = red[lane];
    int a_before = __reduce_add_sync(0xffffffffu, lane < warp ? p.x : 0), e_before = __reduce_add_sync(0xffffffffu, lane < warp ? p.y : 0);
    if (active > 1) {
        const int2 total = make_int2(__reduce_add_sync(0xffffffffu, p.x), __reduce_add_sync(0xffffffffu, p.y));
        if (tid == 0) tally = total;
        cluster_sync();
        int2 c[SEL_MAX_CLUSTER];
#pragma unroll
        for (int r = 0; r < SEL_MAX_CLUSTER; ++r) c[r] = r < rank ? cluster_load2(&tally.x, r) : make_int2(0, 0);
#pragma unroll
        for (int r = 0; r < SEL_MAX_CLUSTER; ++r) {
            a_before += c[r].x;
            e_before += c[r].y;
        }
        cluster_sync();  // a block's tally is read until here
    }
    int at = a_before + min(e_before, left);
    each([&](int j, uint32_t k) {
        unsigned above, equal;
        votes(j, k, above, equal);
        const bool tie = (equal >> lane & 1u) && e_before + __popc(equal & below) < left;  // the lowest of the equals stay
        const unsigned kept = above | __ballot_sync(0xffffffffu, tie);
        if (kept >> lane & 1u) {
            const int r = at + __popc(kept & below);
            idx[r] = j;
            if (out) out[r] = j;
        }
        at += __popc(kept);
        e_before += __popc(equal);
    });
}

// Out of place.  Words: one thread per 16-byte piece of MR kept rows, all loads
// before the first store; the rest (blockIdx.y's last part): one thread per row.
constexpr int MR = 4;
template <int D>
__global__ void __launch_bounds__(256) kv4_move_kernel(const Kv4EvictArgs a, const int* index, const int* count) {
    constexpr int P = D / 32, RB = 256 / P, GR = D / 64;
    const int part = blockIdx.y / a.src.heads, h = blockIdx.y % a.src.heads, b = blockIdx.z, tid = threadIdx.x;
    const size_t bh = (size_t)b * a.src.heads + h;
    pdl_wait();
    pdl_launch_dependents();
    const int n = count[b];
    const int* idx = index + bh * a.keep;
    const size_t s0 = bh * a.src.max_pos, d0 = bh * a.dst.max_pos;
    const int first = blockIdx.x * MR * RB;
    if (part < 2) {
        const int e = tid % P;
        const uint4* sw = reinterpret_cast<const uint4*>(a.src.p[part].w) + s0 * P + e;
        uint4* dw = reinterpret_cast<uint4*>(a.dst.p[part].w) + d0 * P + e;
        int j[MR];
        uint4 v[MR];
#pragma unroll
        for (int i = 0; i < MR; ++i) {
            const int r = first + i * RB + tid / P;
            j[i] = r < n ? idx[r] : -1;
        }
#pragma unroll
        for (int i = 0; i < MR; ++i)
            if (j[i] >= 0) v[i] = __ldcs(sw + (size_t)j[i] * P);
#pragma unroll
        for (int i = 0; i < MR; ++i)
            if (j[i] >= 0) dw[(size_t)(first + i * RB + tid / P) * P] = v[i];
        return;
    }
    if (blockIdx.x == 0 && h == 0 && tid == 0) a.new_len[b] = n;
    for (int r = first + tid; r < min(n, first + MR * RB); r += 256) {
        const size_t sr = s0 + idx[r], dr = d0 + r;
        const float m = a.mass_src[sr];
        if (GR == 2) {
            uint32_t v[4];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                v[2 * w] = reinterpret_cast<const uint32_t*>(a.src.p[w].s)[sr];
                v[2 * w + 1] = reinterpret_cast<const uint32_t*>(a.src.p[w].b)[sr];
            }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                reinterpret_cast<uint32_t*>(a.dst.p[w].s)[dr] = v[2 * w];
                reinterpret_cast<uint32_t*>(a.dst.p[w].b)[dr] = v[2 * w + 1];
            }
        } else {
            const bf16 v0 = a.src.p[0].s[sr], v1 = a.src.p[0].b[sr], v2 = a.src.p[1].s[sr], v3 = a.src.p[1].b[sr];
            a.dst.p[0].s[dr] = v0;
            a.dst.p[0].b[dr] = v1;
            a.dst.p[1].s[dr] = v2;
            a.dst.p[1].b[dr] = v3;
        }
        a.mass_dst[dr] = m;
    }
}

// In place: one block per (sequence, head, K words | V words | the rest) walks
// the kept rows in order, a chunk at a time: read, barrier, write.  index[r] >= r,
// so the rows a chunk overwrites are never read by a later chunk.  MR rows per
// thread and chunk: a chunk costs two memory latencies and two barriers (the case
// above: 35 us, against 24 out of place).
template <int D>
__global__ void __launch_bounds__(1024) kv4_move_inplace_kernel(const Kv4EvictArgs a, const int* index, const int* count) {
    constexpr int P = D / 32, GR = D / 64, RB = 1024 / P;
    const int part = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const size_t bh = (size_t)b * a.src.heads + h;
    pdl_wait();
    pdl_launch_dependents();
    const int n = count[b];
    const int* idx = index + bh * a.keep;
    const size_t row0 = bh * a.src.max_pos;
    if (part == 2 && h == 0 && tid == 0) a.new_len[b] = n;
    if (n == 0 || idx[n - 1] == n - 1) return;  // every row stays where it is
    if (part < 2) {
        uint4* w = reinterpret_cast<uint4*>(a.dst.p[part].w) + row0 * P + tid % P;
        for (int r0 = tid / P; r0 - tid / P < n; r0 += MR * RB) {
            int j[MR];
            uint4 v[MR];
#pragma unroll
            for (int i = 0; i < MR; ++i) j[i] = r0 + i * RB < n ? idx[r0 + i * RB] : -1;
#pragma unroll
            for (int i = 0; i < MR; ++i)
                if (j[i] >= 0) v[i] = w[(size_t)j[i] * P];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < MR; ++i)
                if (j[i] >= 0) w[(size_t)(r0 + i * RB) * P] = v[i];
            __syncthreads();
        }
        return;
    }
    for (int r0 = 0; r0 < n; r0 += 1024) {
        const int r = r0 + tid;
        bf16 v[4 * GR];
        float m = 0.f;
        if (r < n) {
            const size_t sr = row0 + idx[r];
#pragma unroll
            for (int g = 0; g < GR; ++g) {
                v[4 * g] = a.dst.p[0].s[sr * GR + g];
                v[4 * g + 1] = a.dst.p[0].b[sr * GR + g];
                v[4 * g + 2] = a.dst.p[1].s[sr * GR + g];
                v[4 * g + 3] = a.dst.p[1].b[sr * GR + g];
            }
            m = a.mass_dst[sr];
        }
        __syncthreads();
        if (r < n) {
            const size_t dr = row0 + r;
#pragma unroll
            for (int g = 0; g < GR; ++g) {
                a.dst.p[0].s[dr * GR + g] = v[4 * g];
                a.dst.p[0].b[dr * GR + g] = v[4 * g + 1];
                a.dst.p[1].s[dr * GR + g] = v[4 * g + 2];
                a.dst.p[1].b[dr * GR + g] = v[4 * g + 3];
            }
            a.mass_dst[dr] = m;
        }
        __syncthreads();
    }
}

}  // namespace

size_t kv4_evict_scratch_bytes(const Kv4View& src, int keep) {
    return ((size_t)src.batch * src.heads * keep + src.batch) * sizeof(int);
}

cudaError_t launch_kv4_evict(const Kv4EvictArgs& a, void* scratch, cudaStream_t st) {
    int* index = static_cast<int*>(scratch);
    int* count = index + (size_t)a.src.batch * a.src.heads * a.keep;
    // blocks of a head: as many as hold all its positions in shared memory
    int cluster = 1;
    while (cluster < SEL_MAX_CLUSTER && a.src.max_pos > SLICE * cluster) cluster *= 2;
    const int smem = (3 * BINS + std::min(SLICE, (a.src.max_pos + 31) / 32 * 32)) * (int)sizeof(int);
    cudaError_t e = ensure_max_dyn_smem(kv4_select_kernel, (3 * BINS + SLICE) * (int)sizeof(int));
    if (e != cudaSuccess) return e;
    e = launch(kv4_select_kernel, dim3(a.src.heads * cluster, a.src.batch), dim3(SEL_NT), smem, cluster, st, a, cluster, index, count);
    if (e != cudaSuccess) return e;
    const bool wide = a.src.D == 128;
    if (a.dst.p[0].w == a.src.p[0].w) {
        const dim3 grid(3, a.src.heads, a.src.batch);
        return wide ? launch(kv4_move_inplace_kernel<128>, grid, dim3(1024), 0, 1, st, a, (const int*)index, (const int*)count)
                    : launch(kv4_move_inplace_kernel<64>, grid, dim3(1024), 0, 1, st, a, (const int*)index, (const int*)count);
    }
    const int rows = MR * 256 / (a.src.D / 32);
    const dim3 grid((a.keep + rows - 1) / rows, 3 * a.src.heads, a.src.batch);
    return wide ? launch(kv4_move_kernel<128>, grid, dim3(256), 0, 1, st, a, (const int*)index, (const int*)count)
                : launch(kv4_move_kernel<64>, grid, dim3(256), 0, 1, st, a, (const int*)index, (const int*)count);
}

}  // namespace qw
