// Eviction from the 4-bit KV cache by accumulated attention weight.
//
// Per (sequence, kv head) of length n > keep: the last `recent` positions stay,
// and of the others the keep - recent with the largest weight (the lower
// position wins a tie).  The kept rows move to the front in position order,
// with their weights; n <= keep keeps every row.
//
//   1. select: weights become unsigned keys of the same order; a radix select
//      (four 8-bit histogram passes) finds the threshold key and how many of
//      the keys equal to it stay; one ordered pass writes the kept positions.
//   2. move: dst row r = src row index[r].
#include "kv4.h"

namespace qw {
namespace {

constexpr int SEL_NT = 1024;

// Unsigned key of the same order as the float; -0 equals +0, NaN is above everything.
QW_DEV uint32_t order_key(float v) {
    uint32_t u = __float_as_uint(v);
    if (v != v) return 0xFFFFFFFFu;
    if ((u << 1) == 0u) u = 0u;
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

QW_DEV int clamp_len(const Kv4EvictArgs& a, int b) { return max(0, min(a.seq_len[b], a.src.max_pos)); }

// Exclusive prefix of `v` over the block (SEL_NT threads) and the block total.
QW_DEV int block_scan(int v, int* red, int& total) {
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
    if (warp == 0) {
        int t = red[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += u;
        }
        red[lane] = t;
    }
    __syncthreads();
    total = red[31];
    return s - v + (warp ? red[warp - 1] : 0);
}

// index[b][h][0..new length): the kept positions in increasing order.
__global__ void __launch_bounds__(SEL_NT) kv4_select_kernel(const Kv4EvictArgs a, int* index, int* count) {
    __shared__ int hist[256];
    __shared__ int red[32];
    __shared__ int pick[2];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int n = clamp_len(a, b);
    const size_t bh = (size_t)b * a.src.heads + h;
    int* idx = index + bh * a.keep;
    if (tid == 0 && h == 0) count[b] = min(n, a.keep);
    if (n <= a.keep) {
        for (int r = tid; r < a.keep; r += SEL_NT) {
            idx[r] = r < n ? r : -1;
            if (a.index_out) a.index_out[bh * a.keep + r] = r < n ? r : -1;
        }
        return;
    }
    const float* mass = a.mass_src + bh * a.src.max_pos;
    const int old = n - a.recent, want = a.keep - a.recent;
    // threshold key and how many of its equals stay
    uint32_t prefix = 0;
    int left = want;
    if (want > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int j = tid; j < old; j += SEL_NT) {
                const uint32_t k = order_key(mass[j]);
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int acc = 0, d = 255;
                while (d > 0 && acc + hist[d] < left) acc += hist[d--];
                pick[0] = d;
                pick[1] = left - acc;
            }
            __syncthreads();
            prefix |= (uint32_t)pick[0] << shift;
            left = pick[1];
        }
    }
    int base = 0, ties = 0;
    for (int j0 = 0; j0 < n; j0 += SEL_NT) {
        const int j = j0 + tid;
        int above = 0, equal = 0;
        if (j < n) {
            if (j >= old) {
                above = 1;
            } else if (want > 0) {
                const uint32_t k = order_key(mass[j]);
                above = k > prefix;
                equal = k == prefix;
            }
        }
        int tot_eq, tot;
        const int eq_before = ties + block_scan(equal, red, tot_eq);
        const int keep = above | (equal && eq_before < left);
        const int at = base + block_scan(keep, red, tot);
        if (keep) {
            idx[at] = j;
            if (a.index_out) a.index_out[bh * a.keep + at] = j;
        }
        ties += tot_eq;
        base += tot;
    }
}

// Out of place: one thread per (kept row, 16-byte piece of its words).
template <int D>
__global__ void __launch_bounds__(256) kv4_move_kernel(const Kv4EvictArgs a, const int* index, const int* count) {
    constexpr int P = D / 32;  // 16-byte pieces of a packed row
    const int h = blockIdx.y, b = blockIdx.z;
    const size_t bh = (size_t)b * a.src.heads + h;
    const int r = blockIdx.x * (256 / P) + threadIdx.x / P, e = threadIdx.x % P;
    if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.new_len[b] = count[b];
    if (r >= count[b]) return;
    const int j = index[bh * a.keep + r];
    const size_t sr = bh * a.src.max_pos + j, dr = bh * a.dst.max_pos + r;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        reinterpret_cast<uint4*>(a.dst.p[w].w)[dr * P + e] = reinterpret_cast<const uint4*>(a.src.p[w].w)[sr * P + e];
        if (e == 0) {
#pragma unroll
            for (int g = 0; g < D / 64; ++g) {
                a.dst.p[w].s[dr * (D / 64) + g] = a.src.p[w].s[sr * (D / 64) + g];
                a.dst.p[w].b[dr * (D / 64) + g] = a.src.p[w].b[sr * (D / 64) + g];
            }
        }
    }
    if (e == 0) a.mass_dst[dr] = a.mass_src[sr];
}

// In place: one CTA per (sequence, head, K words | V words | the rest) walks the
// kept rows in order, a chunk at a time: read, barrier, write.  index[r] >= r,
// so the rows a chunk overwrites are never read by a later chunk.
template <int D>
__global__ void __launch_bounds__(1024) kv4_move_inplace_kernel(const Kv4EvictArgs a, const int* index, const int* count) {
    constexpr int P = D / 32;
    const int part = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const size_t bh = (size_t)b * a.src.heads + h;
    const int n = count[b];
    const int* idx = index + bh * a.keep;
    const size_t row0 = bh * a.src.max_pos;
    if (part < 2) {
        uint4* w = reinterpret_cast<uint4*>(a.dst.p[part].w) + row0 * P;
        for (int r0 = 0; r0 < n; r0 += 1024 / P) {
            const int r = r0 + tid / P, e = tid % P;
            uint4 v;
            if (r < n) v = w[(size_t)idx[r] * P + e];
            __syncthreads();
            if (r < n) w[(size_t)r * P + e] = v;
            __syncthreads();
        }
        return;
    }
    if (h == 0 && tid == 0) a.new_len[b] = n;
    for (int r0 = 0; r0 < n; r0 += 1024) {
        const int r = r0 + tid;
        bf16 v[4 * (D / 64)];
        float m = 0.f;
        if (r < n) {
            const size_t sr = row0 + idx[r];
#pragma unroll
            for (int g = 0; g < D / 64; ++g) {
                v[4 * g] = a.dst.p[0].s[sr * (D / 64) + g];
                v[4 * g + 1] = a.dst.p[0].b[sr * (D / 64) + g];
                v[4 * g + 2] = a.dst.p[1].s[sr * (D / 64) + g];
                v[4 * g + 3] = a.dst.p[1].b[sr * (D / 64) + g];
            }
            m = a.mass_dst[sr];
        }
        __syncthreads();
        if (r < n) {
            const size_t dr = row0 + r;
#pragma unroll
            for (int g = 0; g < D / 64; ++g) {
                a.dst.p[0].s[dr * (D / 64) + g] = v[4 * g];
                a.dst.p[0].b[dr * (D / 64) + g] = v[4 * g + 1];
                a.dst.p[1].s[dr * (D / 64) + g] = v[4 * g + 2];
                a.dst.p[1].b[dr * (D / 64) + g] = v[4 * g + 3];
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
    const int D = a.src.D;
    kv4_select_kernel<<<dim3(a.src.heads, a.src.batch), SEL_NT, 0, st>>>(a, index, count);
    if (a.dst.p[0].w == a.src.p[0].w) {
        const dim3 grid(3, a.src.heads, a.src.batch);
        if (D == 128)
            kv4_move_inplace_kernel<128><<<grid, 1024, 0, st>>>(a, index, count);
        else
            kv4_move_inplace_kernel<64><<<grid, 1024, 0, st>>>(a, index, count);
    } else {
        const int rows = 256 / (D / 32);
        const dim3 grid((a.keep + rows - 1) / rows, a.src.heads, a.src.batch);
        if (D == 128)
            kv4_move_kernel<128><<<grid, 256, 0, st>>>(a, index, count);
        else
            kv4_move_kernel<64><<<grid, 256, 0, st>>>(a, index, count);
    }
    return cudaGetLastError();
}

}  // namespace qw
