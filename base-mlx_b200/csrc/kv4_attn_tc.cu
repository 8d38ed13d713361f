// Attention over the 4-bit KV cache for many rows per kv head (prompt chunks),
// on the tcgen05 tensor cores.
//
// A thread block takes NB = 1 or 2 blocks of 128 columns (row, query head) of one
// (sequence, kv head) and walks the keys they see in tiles of 128.  A key's
// element in group g is s_g (n - 8) + c_g with c_g = b_g + 8 s_g:
//   S  = Q K'^T + Q* C*^T    K' = s (n - 8): an 8-bit by a 3-bit number, exact in
//                            fp16; Q exact in fp16 (scaled per column as in
//                            kv4_tile.cuh); Q* and C* hold the group sums of q and
//                            the c_g in pieces of 11 bits, one more k-step of 16
//   x  = c S - m             fp32, two threads per column
//   P  = 2^x                 fp16 in TMEM, over the first half of S
//   O += P V                 V dequantised to fp16, fp32 sums in TMEM
// So scores are exact up to fp32 sums, and the softmax threads need no per-key
// numbers.  (With the integers themselves as operand and a sum per group, the
// per-key scales cost four shared-memory words per score, and their reads were
// the bound: 309 us for 1024 rows of 32 heads on 8192 keys.)  K and V are taken
// times powers of two that put the block's largest value (found first, from
// scales and biases alone) where fp16 holds it; the running maximum moves only
// when a score passes it by 2^8 (P <= 2^15), and then O is rescaled in TMEM.
//
// 1024 rows of 32 heads on 8192 keys (8 kv heads): 188 us = 0.41 of the tensor
// rate.  A tile of 128 keys takes 5900 cycles for 256 columns, of which the
// products need 2200 and the powers 2050; the softmax threads are busy
// throughout: 2700 cycles in the softmax, 1500 expanding, 650 issuing loads.
//
// Roles: one lane of the last warp issues the products; all other warps, two
// threads per column with half a tile's keys each, do the softmax and between two
// softmaxes expand a share of packed rows (the values of the next tile, the keys
// of the one after), which they loaded into registers a tile earlier.  With NB =
// 2 one column block's softmax runs beside the other's products.  (Three warps of
// their own for the expansion took 11 400 cycles a tile: alone on their issue
// slots they run at the pace of instruction fetch and of single dependent
// chains.)  Every wait is bounded: a lost arrival sets QW_DERR_TIMEOUT and the
// block still frees its TMEM and ends.
#include "kv4_join.cuh"
#include "kv4_launch.h"
#include "kv4_tc.h"
#include "kv4_tcgen.cuh"
#include "smem_attr.h"

namespace qw {
namespace {

using namespace kv4;

template <int NB>
constexpr int THREADS = 256 * NB + 32;
constexpr float BASE = 7.f;           // P = 2^(x - max + 7): normal fp16 numbers down to 2^-21 of the largest
constexpr float RAISE = BASE + 8.f;   // a larger exponent raises the maximum
constexpr float UNSET = -3.0e38f;

// Shared memory, from a 1 KB aligned base.
template <int D, int NB>
struct Plan {
    static constexpr int GR = D / 64;
    static constexpr int QB = q_block_bytes(D), KB = GR * KT * 128 + KT * 32, VB = GR * KT * 128;
    static constexpr int Q = 5120;           // after the barriers and two exchange arrays: [NB]{[GR][128 rows][128 B] swizzled; Q*}
    static constexpr int K = Q + NB * QB;    // [2]{[GR][128 keys][128 B] swizzled; C*}
    static constexpr int V = K + 2 * KB;     // [2][GR][128 keys][128 B], swizzled, read along the keys
    static constexpr int BYTES = V + 2 * VB + 1024;
    // TMEM columns of a column block: S (P over its first half), O
    static constexpr uint32_t TO = KT, TB = KT + D, TMEM = NB * TB <= 256 ? 256 : 512;
};

QW_DEV float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <int D, int NB>
__global__ void __launch_bounds__(THREADS<NB>, 1) kv4_attn_tc_kernel(const Kv4AttnArgs a, int ncb, int nsplit, float* part, float2* pml,
                                                                        unsigned char* qkeep) {
    using P = Plan<D, NB>;
    constexpr int GR = P::GR, CB = CM * NB, PW0 = 8 * NB;  // columns of the block, first producer warp
    extern __shared__ unsigned char tc_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)tc_raw + 1023) & ~(uintptr_t)1023);
    // barriers: tile i uses [i & 1] of the paired ones; those per column block count tiles
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sm);  // K operand written
    uint64_t* k_free = k_full + 2;                        // products Q N of every column block done
    uint64_t* v_full = k_free + 2;
    uint64_t* v_free = v_full + 2;
    uint64_t* s_full = v_free + 2;                        // per column block: scores in TMEM
    uint64_t* p_full = s_full + 2;
    uint64_t* pv_done = p_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);
    float* kvmax = reinterpret_cast<float*>(tmem_slot + 2);  // [8 NB][2] of the warps: largest |K|, |V|
    int* left_out = reinterpret_cast<int*>(kvmax + 16 * NB);  // first key whose V is left out (see partial)
    float* xch = reinterpret_cast<float*>(sm + 1024);       // [round][half][CB]: largest scores; in the end the halves' sums
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_wait();
    pdl_launch_dependents();

    // heaviest column blocks first
    const int per_cb = nsplit * a.c.heads * a.c.batch;
    const int cb = ncb - 1 - (int)(blockIdx.x / per_cb), rest = (int)(blockIdx.x % per_cb);
    const int sp = rest % nsplit, h = rest / nsplit % a.c.heads, b = rest / nsplit / a.c.heads;
    const int G = a.Hq / a.c.heads, C = G * a.S;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, a.err, tid == 0 && cb == 0 && sp == 0 && h == 0);
    const int T = rw.off + rw.n;
    // rows of the block's columns, keys they see, this split's tiles
    const int i_first = cb * CB / G, i_last = min(rw.n, (min(C, (cb + 1) * CB) - 1) / G + 1) - 1;
    const int keys = i_last < i_first ? 0 : a.causal ? min(T, rw.off + i_last + 1) : T;
    const int nt = (keys + KT - 1) / KT, t0 = nt * sp / nsplit, t1 = nt * (sp + 1) / nsplit;  // (nt < 2^24, nsplit <= 64)
    const int all = a.causal ? min(T, rw.off + i_first + 1) : T;  // keys that every column sees
    const size_t seg = ((size_t)b * a.c.heads + h) * ncb + cb;

    const int half = (warp >> 2) & 1;  // softmax threads: half of a tile's keys
    const int col = min((warp >> 3) * CM + (tid & 127), CB - 1), c = cb * CB + col, i_row = c / G, head = h * G + c % G;
    const bool row = c < C && i_row < rw.n;
    // (worked out where they are used: between the block's begin and end registers are short)
    auto out_row = [&] {
        const int i = c / G;
        return a.out + (b * a.os.b + (long long)i * a.os.s + (long long)(h * G + (c - i * G)) * a.os.h);
    };
    auto lse_at = [&] { return a.lse + (((size_t)b * a.S + c / G) * a.Hq + h * G + c % G); };
    if (t0 == t1) {  // nothing to see: zeros (a split's empty share is skipped by the joining kernel)
        if (nsplit == 1 && warp < PW0 && half == 0 && c < C) {
            for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(out_row() + d) = make_uint4(0u, 0u, 0u, 0u);
            if (a.lse) *lse_at() = -INFINITY;
        }
        return;
    }
    if (tid == 0) {
        *left_out = 0x7FFFFFFF;
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + i, 256 * NB);
            mbar_init(k_free + i, 1);
            mbar_init(v_full + i, 256 * NB);
            mbar_init(v_free + i, 1);
            mbar_init(s_full + i, 1);
            mbar_init(p_full + i, 256);
            mbar_init(pv_done + i, 1);
        }
        fence_mbar_init();
    }
    if (warp == PW0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(P::TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    // the two warps that share 32 columns meet
    auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(2 + (warp >> 3) * 4 + (warp & 3)) : "memory"); };
    auto pair_any = [&](bool v) {
        uint32_t r;
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %2, 0;\n\tbarrier.cta.red.or.pred q, %1, 64, p;\n\tselp.b32 %0, 1, 0, q;\n\t}\n"
            : "=r"(r)
            : "r"(2 + (warp >> 3) * 4 + (warp & 3)), "r"((int)v)
            : "memory");
        return r != 0;
    };
    const Rows rows = head_rows<D>(a.c, (size_t)b * a.c.heads + h);
    const int key_end = min(T, t1 * KT);  // this block's keys end here
    const int n_tiles = t1 - t0;
    // Expansion: a thread takes 16-byte pieces (4 words of a row), thread after thread.
    constexpr int CPR = D / 32, PIECES = KT * CPR, NTH = 256 * NB, PER = PIECES >= NTH ? PIECES / NTH : 1;
    const bool has_piece = tid < PIECES;  // D = 64 and two column blocks: half of the threads
    struct Share {
        uint4 w[PER];
        uint16_t s[PER], z[PER];  // scale and bias of the piece's group
    } ks, vs;
    uint32_t cs = 0, cz = 0;  // threads 0 .. 127: scales and biases of one key of the tile, every group
    // A block-wide base and a 32-bit offset of the thread's own each.
    const uint32_t po = (uint32_t)tid, so = (uint32_t)(tid / CPR * GR + ((tid % CPR) >> 1));
    constexpr uint32_t PSTEP = NTH, SSTEP = NTH / CPR * GR;
    auto load = [&](Share& x, int which, int i) {  // zeros past the last key
        const int k0 = (t0 + i) * KT;
        const uint4* src = reinterpret_cast<const uint4*>(rows.w[which] + (size_t)k0 * (D / 2));
        const uint16_t* s = reinterpret_cast<const uint16_t*>(rows.s[which]) + (size_t)k0 * GR;
        const uint16_t* z = reinterpret_cast<const uint16_t*>(rows.b[which]) + (size_t)k0 * GR;
        if (k0 + KT <= T && (PIECES >= NTH || has_piece)) {
#pragma unroll
            for (uint32_t j = 0; j < PER; ++j) {
                x.w[j] = src[po + PSTEP * j];
                x.s[j] = s[so + SSTEP * j];
                if (which) x.z[j] = z[so + SSTEP * j];
            }
            return;
        }
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const bool in = has_piece && k0 + (tid + NTH * (int)j) / CPR < T;
            x.w[j] = in ? src[po + PSTEP * j] : make_uint4(0u, 0u, 0u, 0u);
            x.s[j] = in ? s[so + SSTEP * j] : (uint16_t)0;
            if (which) x.z[j] = in ? z[so + SSTEP * j] : (uint16_t)0;
        }
    };
    auto load_k = [&](int i) {
        if (i >= n_tiles) return;
        load(ks, 0, i);
        const int key = (t0 + i) * KT + tid;
        cs = tid < KT && key < T ? group_pair<GR>(rows.s[0], key) : 0u;
        cz = tid < KT && key < T ? group_pair<GR>(rows.b[0], key) : 0u;
    };
    auto load_v = [&](int i) {
        if (i < n_tiles) load(vs, 1, i);
    };
    float cc = 0.f;  // score of a column = cc * S (softmax threads; K's power of two comes in below)
    if (warp < PW0) {
        // Q operand: column `col`, the thread's half of its chunks, elements in the order of an expanded word.  Everything
        // that the block begins with is on its way at once: the queries, the first tile's rows, the scales and biases.
        // (The queries come row by row into their places, to be converted there: a row per lane is 32 lines a load, which
        // alone took 4000 cycles.)
        constexpr int QW = 4 * GR;  // chunks of a thread: with two groups one of them
        auto all_sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(256 * NB) : "memory"); };
        long long* off = reinterpret_cast<long long*>(xch);  // [CB]
        if (half == 0) off[col] = row ? b * a.qs.b + (long long)i_row * a.qs.s + (long long)head * a.qs.h : -1;
        load_k(0);
        load_v(0);
        all_sync();
#pragma unroll
        for (int j = 0; j < QW; ++j) {
            const int p = tid + 256 * NB * j, qc = p / (D / 8), k = p % (D / 8);
            const long long o = off[qc];
            cp_async16_zfill(smem_u32(sm + P::Q + (qc >> 7) * P::QB + (k >> 3) * CM * 128 + chunk_at(qc & 127, k & 7)),
                       o < 0 ? a.q : a.q + o + 8 * k, o >= 0);
        }
        cp_async_commit();
        // largest magnitudes that the block's rows can stand for: max(|b|, |b + 15 s|)
        constexpr int KW = 2 / GR;  // keys of a 32-bit word of scales (rows end at a multiple of 16)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            float mx = 0.f;
            const uint32_t* s = reinterpret_cast<const uint32_t*>(rows.s[v]);
            const uint32_t* z = reinterpret_cast<const uint32_t*>(rows.b[v]);
#pragma unroll 4
            for (int w = t0 * KT / KW + tid; w < (key_end + KW - 1) / KW; w += 256 * NB) {
                const uint32_t us = s[w], uz = z[w];
                mx = fmaxf(mx, reach(bits_lo_f(us), bits_lo_f(uz)));
                if (GR == 2 || w * KW + 1 < key_end) mx = fmaxf(mx, reach(bits_hi_f(us), bits_hi_f(uz)));
            }
            mx = warp_max(mx);
            if (lane == 0) kvmax[2 * warp + v] = mx;
        }
        cp_async_wait<0>();
        all_sync();
        unsigned char* qo = sm + P::Q + (col >> 7) * P::QB;
        auto mine = [&](int k) { return reinterpret_cast<uint4*>(qo + (half * QW + k) / 8 * CM * 128 + chunk_at(col & 127, (half * QW + k) % 8)); };
        float mx = 0.f, sum = 0.f;
#pragma unroll 2
        for (int k = 0; k < QW; ++k) {
            const uint4 raw = *mine(k);
            const uint32_t X[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float lo = bits_lo_f(X[e]), hi = bits_hi_f(X[e]);
                sum += lo + hi;
                mx = fmaxf(mx, fmaxf(fabsf(lo), fabsf(hi)));
            }
        }
        xch[half * CB + col] = mx;
        xch[(2 + half) * CB + col] = sum;
        pair_sync();
        mx = fmaxf(xch[col], xch[CB + col]);
        const int ex = max((int)(__float_as_uint(mx) >> 23) - 127, -100);
        const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
        cc = ldexpf(a.scale * LOG2E, ex - 14);
#pragma unroll 2
        for (int j = 0; j < QW; ++j) {
            const uint4 raw = *mine(j);
            const uint32_t X[4] = {raw.x, raw.y, raw.z, raw.w};
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[2 * e] = bits_lo_f(X[e]) * up;
                x[2 * e + 1] = bits_hi_f(X[e]) * up;
            }
            *mine(j) = make_uint4(h2(x[0], x[4]), h2(x[1], x[5]), h2(x[2], x[6]), h2(x[3], x[7]));
        }
        // Q*: a group's sum times 2^-6 in three fp16 terms, k = 5 g + {0..4}: hi, hi, mid, mid, lo
        // (against the two terms of 2^6 c: hi, lo, hi, lo, hi)
        if (half == 0) {
            __half t[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) t[e] = __float2half_rn(0.f);
#pragma unroll
            for (int g = 0; g < GR; ++g) {
                const float s = GR == 2 ? xch[(2 + g) * CB + col] : xch[2 * CB + col] + xch[3 * CB + col];
                const float v = s * up * 0.015625f;
                const __half hi = __float2half_rn(v), mid = __float2half_rn(v - __half2float(hi));
                t[5 * g] = t[5 * g + 1] = hi;
                t[5 * g + 2] = t[5 * g + 3] = mid;
                t[5 * g + 4] = __float2half_rn(v - __half2float(hi) - __half2float(mid));
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t r[4];
#pragma unroll
                for (int f = 0; f < 4; ++f) r[f] = as_u(__halves2half2(t[8 * e + 2 * f], t[8 * e + 2 * f + 1]));
                *reinterpret_cast<uint4*>(qo + GR * CM * 128 + at16(col & 127, e)) = make_uint4(r[0], r[1], r[2], r[3]);
            }
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (qkeep && sp == nsplit - 1) {  // (the last split of a block with rows has tiles)
        uint4* dst = reinterpret_cast<uint4*>(qkeep + seg * NB * P::QB);
        for (int p = tid; p < NB * P::QB / 16; p += THREADS<NB>) dst[p] = reinterpret_cast<const uint4*>(sm + P::Q)[p];
        if (warp < PW0 && half == 0)
            reinterpret_cast<float*>(qkeep + (size_t)a.c.batch * a.c.heads * ncb * NB * P::QB)[seg * CB + col] = cc;
    }
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    // exponents of the largest values
    auto exponent = [&](int v) {
        float m = 0.f;
#pragma unroll
        for (int w = 0; w < PW0; ++w) m = fmaxf(m, kvmax[2 * w + v]);
        return top_exponent(m);
    };
    const int ek = exponent(0), ev = exponent(1);
    bool ok = true;

    if (warp < PW0) {
        // ---- softmax: two threads per column, half of a tile's keys each ----------------------------------
        constexpr int KH = 32;  // keys of a thread and round
        const int blk = warp >> 3;
        const uint32_t tm = tmem + blk * P::TB + ((uint32_t)(32 * (warp & 3)) << 16);
        const int vis = row ? (a.causal ? min(T, rw.off + i_row + 1) : T) : 0;
        cc = ldexpf(cc, ek - 7);
        const unsigned long long c2 = pack2(cc, cc);

        // ---- expansion of this thread's share of a tile --------------------------------------------------
        const float kup = __uint_as_float((uint32_t)(127 + 7 - ek) << 23), vup = __uint_as_float((uint32_t)(127 + 16 - ev) << 23);
        // A NaN in V: where every column sees the key its value is simply NaN; in a tile that some column sees in
        // part only, the value is left out and the outputs of the columns that see the first such key become NaN in the end.
        auto partial = [&](int i) { return (t0 + i + 1) * KT > all; };
        auto store_k = [&](int i) {  // tile i's K operand from ks, cs, cz
            if (i >= n_tiles) return;
            if (ok && i > 1 && !wait_bar(k_free + (i & 1), ((i - 2) >> 1) & 1)) ok = false;
            unsigned char* dst = sm + P::K + (i & 1) * P::KB;
            if (has_piece)
#pragma unroll
                for (int j = 0; j < PER; ++j) expand_piece<D>(ks.w[j], tid + NTH * j, dst, Centred(u16_to_f(ks.s[j]) * kup));
            if (tid < KT) {
                const int key = (t0 + i) * KT + tid;
                if (partial(i) && key < T) {
                    const uint32_t s = group_pair<GR>(rows.s[1], key), z = group_pair<GR>(rows.b[1], key);
                    if (!finite(bits_lo_f(s), bits_lo_f(z)) || !finite(bits_hi_f(s), bits_hi_f(z))) atomicMin(left_out, key);
                }
                store_offsets<GR>(dst + GR * KT * 128, tid, cs, cz, kup);
            }
        };
        auto store_v = [&](int i) {
            if (i >= n_tiles) return;
            if (ok && i > 1 && !wait_bar(v_free + (i & 1), ((i - 2) >> 1) & 1)) ok = false;
            unsigned char* dst = sm + P::V + (i & 1) * P::VB;
            if (has_piece)
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    float s = u16_to_f(vs.s[j]), z = u16_to_f(vs.z[j]);
                    if (partial(i) && !finite(s, z)) s = z = 0.f;
                    // n 2^-18 times 2^18 s plus z, times 2^(-2 - ev): s is at most 2/15 of the largest value
                    const __half2 s2 = __float2half2_rn(s * vup), z2 = __float2half2_rn(z * vup * 0x1p-18f);
                    expand_piece<D>(vs.w[j], tid + NTH * j, dst, [&](uint32_t n) { return as_u(__hfma2(as_h2(n), s2, z2)); });
                }
        };
        // Stores first, then one fence, then the loads: a fence waits for the thread's loads in flight.
        auto publish = [&](int ik, int iv) {
            fence_proxy_async_smem();
            if (iv < n_tiles) arrive(v_full + (iv & 1));
            if (ik < n_tiles) arrive(k_full + (ik & 1));
        };
        store_k(0);
        store_v(0);
        publish(0, 0);  // and the Q operand
        load_k(1);
        load_v(1);
        store_k(1);
        publish(1, n_tiles);
        load_k(2);

        float nm = 0.f, l = 0.f, thr = UNSET;  // BASE - maximum; up to thr the maximum stays
        for (int i = 0; i < n_tiles; ++i) {
            if (ok && !wait_bar(s_full + blk, i & 1)) ok = false;
            fence_after();
            // Two rounds of 64 keys, 32 of them this thread's.  P of a round lies over columns of S that this
            // round or the one before has read; the two warps of the column meet after each read, and hear
            // whether either of them met a larger score.
#pragma unroll 1
            for (int m = 0; m < 2; ++m) {
                const int k0 = 64 * m + 32 * half, key0 = (t0 + i) * KT + k0;
                const unsigned long long nm2 = pack2(nm, nm);
                float x[KH];
                ld16(tm + k0, *reinterpret_cast<float(*)[16]>(&x[0]));
                ld16(tm + k0 + 16, *reinterpret_cast<float(*)[16]>(&x[16]));
                wait_ld();
#pragma unroll
                for (int k = 0; k < KH; k += 2) unpack2(fma2(c2, pack2(x[k], x[k + 1]), nm2), x[k], x[k + 1]);
                if (key0 + KH > all)
#pragma unroll
                    for (int k = 0; k < KH; ++k)
                        if (key0 + k >= vis) x[k] = -INFINITY;
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < KH; k += 2) top = max3(top, x[k], x[k + 1]);
                if (pair_any(top > thr)) {
                    wait_st();  // P of the round before and O of a raise there are read back below
                    xch[(2 * m + half) * CB + col] = top;
                    pair_sync();
                    top = fmaxf(top, xch[(2 * m + (half ^ 1)) * CB + col]);
                    // raise the maximum of the columns that ask for it, and rescale what they have summed
                    float al = 1.f;
                    if (top > thr) {
                        const float up = BASE - top;
                        al = thr == UNSET ? 0.f : ex2(up);  // the column's first key: nothing summed so far
                        nm += up;
                        thr = RAISE;
#pragma unroll
                        for (int k = 0; k < KH; ++k) x[k] += up;
                    }
                    if (i > 0)  // P V of the tile before is complete: the products of this one came after it
#pragma unroll 1
                        for (int d = half * (D / 2); d < (half + 1) * (D / 2); d += 16) {
                            float o[16];
                            uint32_t r[16];
                            ld16(tm + P::TO + d, o);
                            wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(o[e] * al);
                            st16(tm + P::TO + d, r);
                        }
                    if (m > 0) {  // this tile's first round
                        float o[16];
                        uint32_t r[16];
                        ld16(tm + half * (KH / 2), o);
                        wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float2 f = __half22float2(as_h2(__float_as_uint(o[e])));
                            r[e] = h2(f.x * al, f.y * al);
                        }
                        st16(tm + half * (KH / 2), r);
                    }
                    l *= al;
                }
                unsigned long long l2[2] = {0ull, 0ull};
                uint32_t r[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float p0 = ex2(x[2 * e]), p1 = ex2(x[2 * e + 1]);
                    l2[e & 1] = add2(l2[e & 1], pack2(p0, p1));
                    r[e] = h2(p0, p1);
                }
                st16(tm + k0 / 2, r);
                float l0, l1;
                unpack2(add2(l2[0], l2[1]), l0, l1);
                l += l0 + l1;
            }
            wait_st();
            fence_before();
            arrive(p_full + blk);
            store_v(i + 1);
            store_k(i + 2);
            publish(i + 2, i + 1);
            load_v(i + 2);
            load_k(i + 3);
        }
        xch[half * CB + col] = l;
        pair_sync();
        l = xch[col] + xch[CB + col];
        if (ok && !wait_bar(pv_done + blk, (n_tiles - 1) & 1)) ok = false;
        fence_after();
        // ---- output ---------------------------------------------------------------------------------
        const bool has = row && l != 0.f;
        if (ok && !wait_bar(k_full + ((n_tiles - 1) & 1), ((n_tiles - 1) >> 1) & 1)) ok = false;  // complete: it shows left_out
        const bool spoilt = row && *left_out < (a.causal ? rw.off + i_row + 1 : T);
        // A split leaves its sums as they are, below 2^16 V a key: with V past 2^70 its share is taken 2^drop smaller, output and
        // sum alike, against a base as much larger, so that they stay in range.
        const int drop = nsplit == 1 ? 0 : max(0, ev - 70);
        const float less = __uint_as_float((uint32_t)(127 - drop) << 23);
        const float f = spoilt ? __int_as_float(0x7FC00000) : nsplit == 1 ? (has ? 1.f / l : 0.f) : less;
        const float e0 = 4.f, e1 = __uint_as_float((uint32_t)(127 + ev) << 23);
        const size_t slot = (seg * nsplit + sp) * CB + col;
        // Through shared memory (the Q and K operands, of which every product is done), so that lanes write along
        // rows: [32 columns][128 B], swizzled.
        const bf16* out = out_row();
        unsigned char* stage = sm + P::Q + warp * 4096;
        auto piece = [&](int r, int ch) { return reinterpret_cast<uint4*>(stage + chunk_at(r, ch)); };
        const int c_warp = cb * CB + (warp >> 3) * CM + 32 * (warp & 3);  // the warp's first column
        constexpr int STEP = D / 2 < 32 ? D / 2 : 32;
#pragma unroll 1
        for (int d0 = half * (D / 2); d0 < (half + 1) * (D / 2); d0 += nsplit == 1 ? D / 2 : STEP) {
#pragma unroll 1
            for (int d = 0; d < (nsplit == 1 ? D / 2 : STEP); d += 16) {
                float o[16];
                ld16(tm + P::TO + d0 + d, o);
                wait_ld();
#pragma unroll
                for (int g = 0; g < 16; g += 8) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = o[g + (e < 4 ? 2 * e : 2 * e - 7)] * f * e0 * e1;  // columns hold 0, 4, 1, 5, ...
                    if (nsplit == 1) {
                        *piece(lane, (d + g) / 8) =
                            has ? make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]))
                                : make_uint4(0u, 0u, 0u, 0u);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e += 4)
                            *piece(lane, (d + g + e) / 4) =
                                make_uint4(__float_as_uint(v[e]), __float_as_uint(v[e + 1]), __float_as_uint(v[e + 2]), __float_as_uint(v[e + 3]));
                    }
                }
            }
            __syncwarp();
            if (nsplit == 1) {
                constexpr int NCH = D / 16;  // 16-byte chunks of a row's half
#pragma unroll
                for (int it = 0; it < NCH; ++it) {
                    const int r = it * (32 / NCH) + lane / NCH, ch = lane % NCH;
                    bf16* dst = reinterpret_cast<bf16*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), r));
                    if (ok && c_warp + r < C) *reinterpret_cast<uint4*>(dst + d0 + 8 * ch) = *piece(r, ch);
                }
            } else {
                constexpr int NCH = STEP / 4;
#pragma unroll
                for (int it = 0; it < NCH; ++it) {
                    const int r = it * (32 / NCH) + lane / NCH, ch = lane % NCH;
                    if (ok && c_warp + r < C) *reinterpret_cast<uint4*>(part + (slot - lane + r) * D + d0 + 4 * ch) = *piece(r, ch);
                }
            }
            __syncwarp();
        }
        if (ok && c < C && half == 0) {
            if (nsplit == 1) {
                if (a.lse) *lse_at() = has ? (log2f(l) - nm) * LN2 : -INFINITY;
            } else {
                pml[slot] = make_float2(l != 0.f ? (float)drop - nm : M0, l * less);
            }
        }
    } else {
        // ---- products ------------------------------------------------------------------------------------
        const uint32_t qa = smem_u32(sm + P::Q), ka = smem_u32(sm + P::K);
        const uint64_t qd = desc(qa, 16), kd = desc(ka, 16), vd = desc(smem_u32(sm + P::V), KT * 128);
        const uint64_t qx = desc16(qa + GR * CM * 128), kx = desc16(ka + GR * KT * 128);
        // descriptor of an operand `bytes` further on (shared addresses stay below the field's end)
        auto at = [](uint64_t d, uint32_t bytes) { return d + (bytes >> 4); };
        auto scores = [&](int blk, int i) {  // S of tile i
            const uint32_t qo = blk * P::QB, ko = (i & 1) * P::KB, d = tmem + blk * P::TB;
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                mma_ss(d, at(qd, qo + (k >> 2) * CM * 128 + 32 * (k & 3)), at(kd, ko + (k >> 2) * KT * 128 + 32 * (k & 3)), idesc(KT, false),
                       k != 0 ? 1u : 0u);
            mma_ss(d, at(qx, qo), at(kx, ko), idesc(KT, false), 1u);
            commit(s_full + blk);
            if (blk == NB - 1) commit(k_free + (i & 1));
        };
        if (!wait_bar(k_full, 0)) ok = false;
        if (ok) {
            fence_after();
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) scores(blk, 0);
        }
        for (int i = 0; i < n_tiles && ok; ++i) {
            if (!wait_bar(v_full + (i & 1), (i >> 1) & 1)) ok = false;
            const uint32_t vo = (i & 1) * P::VB;
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
                if (ok && !wait_bar(p_full + blk, i & 1)) ok = false;
                if (!ok) break;
                fence_after();
#pragma unroll
                for (int k = 0; k < KT / 16; ++k)
                    mma_ts(tmem + blk * P::TB + P::TO, tmem + blk * P::TB + 8 * k, at(vd, vo + 16 * 128 * k), idesc(D, true),
                           (i | k) != 0 ? 1u : 0u);
                commit(pv_done + blk);
                if (blk == NB - 1) commit(v_free + (i & 1));
                if (i + 1 < n_tiles) {  // S holds P until its product is done
                    if ((blk == 0 && !wait_bar(k_full + ((i + 1) & 1), ((i + 1) >> 1) & 1)) || !wait_bar(pv_done + blk, i & 1)) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    scores(blk, i + 1);
                }
            }
        }
        ok = __all_sync(0xffffffffu, ok);
    }
    if (!ok && a.err) atomicOr(a.err, (int)QW_DERR_TIMEOUT);
    fence_before();
    __syncthreads();
    if (warp == PW0) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::TMEM) : "memory");
    }
}

// Joins the splits' partials.  One warp per row, the rows of a sequence in order.
constexpr int JOIN_WARPS = 4;
template <int D>
__global__ void __launch_bounds__(32 * JOIN_WARPS) kv4_attn_tc_join_kernel(const Kv4AttnArgs a, int cb_size, int ncb, int nsplit,
                                                                           const float* part, const float2* pml) {
    const int b = blockIdx.y, G = a.Hq / a.c.heads, lane = threadIdx.x & 31;
    const int item = blockIdx.x * JOIN_WARPS + (threadIdx.x >> 5), h = item % a.Hq, i = item / a.Hq;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, nullptr, false);
    if (i >= a.S) {
        pdl_wait();
        return;
    }
    const int c = i * G + h % G, cb = c / cb_size, C = G * a.S;
    const int i_last = min(rw.n, (min(C, (cb + 1) * cb_size) - 1) / G + 1) - 1;
    const int T = rw.off + rw.n, nt = ((a.causal ? min(T, rw.off + i_last + 1) : T) + KT - 1) / KT;
    bf16* dst = a.out + (b * a.os.b + (long long)i * a.os.s + (long long)h * a.os.h);
    float* lse = a.lse ? a.lse + ((size_t)b * a.S + i) * a.Hq + h : nullptr;
    const size_t s0 = ((((size_t)b * a.c.heads + h / G) * ncb + cb) * nsplit) * cb_size + c % cb_size;
    pdl_wait();
    pdl_launch_dependents();  // the weights kernel expands its keys meanwhile
    if (i >= rw.n) {
        if (lane < D / 8) *reinterpret_cast<uint4*>(dst + 8 * lane) = make_uint4(0u, 0u, 0u, 0u);
        if (lse && lane == 0) *lse = -INFINITY;
        return;
    }
    // a split without tiles has left nothing
    auto slot = [&](int k) {
        return nt * k / nsplit == nt * (k + 1) / nsplit ? -1ll : (long long)(s0 + (size_t)k * cb_size);
    };
    join_row<D, 1, 4>(nsplit, 0, slot, part, pml, nullptr, dst, lse);
}

template <int D, int NB>
cudaError_t launch_tc(const Kv4AttnArgs& a, const TcShape& sp, float* part, float2* ml, unsigned char* qkeep, cudaStream_t st) {
    constexpr int smem = Plan<D, NB>::BYTES;
    cudaError_t e = ensure_max_dyn_smem(kv4_attn_tc_kernel<D, NB>, smem);
    if (e != cudaSuccess) return e;
    const long long blocks = (long long)sp.ncb * sp.nsplit * a.c.heads * a.c.batch;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
    e = launch(kv4_attn_tc_kernel<D, NB>, dim3((unsigned)blocks), dim3(THREADS<NB>), smem, 1, st, a, sp.ncb, sp.nsplit, part, ml,
               qkeep);
    if (e != cudaSuccess || sp.nsplit == 1) return e;
    return launch(kv4_attn_tc_join_kernel<D>, dim3((unsigned)((a.S * (long long)a.Hq + JOIN_WARPS - 1) / JOIN_WARPS), a.c.batch), dim3(32 * JOIN_WARPS), 0, 1, st, a, CM * NB, sp.ncb,
                  sp.nsplit, (const float*)part, (const float2*)ml);
}

}  // namespace

TcShape kv4_tc_shape(const Kv4View& c, int S, int Hq, int num_sms) {
    const long long C = (long long)(Hq / c.heads) * S;
    TcShape s;
    s.nb = C > CM ? 2 : 1;
    s.ncb = (int)((C + CM * s.nb - 1) / (CM * s.nb));
    // splits of the keys: fill rounds of one block per SM, at least two tiles each if the cache were
    // full; a split costs a partial's write and read, counted as a tenth of a round
    const long long segs = (long long)s.ncb * c.heads * c.batch;
    s.nsplit = 1;
    float best = 1e30f;
    for (int n = 1; n <= 64 && (n == 1 || n * 2 * KT <= c.max_pos); ++n) {
        const float t = (float)((segs * n + num_sms - 1) / num_sms) / n * (1.f + 0.1f * (n - 1));
        if (t < best) {
            best = t;
            s.nsplit = n;
        }
    }
    s.part_rows = s.nsplit > 1 ? (size_t)segs * s.nsplit * CM * s.nb : 0;
    s.kept_bytes = (size_t)segs * s.nb * (q_block_bytes(c.D) + CM * 4);
    return s;
}

cudaError_t launch_kv4_attn_tc(const Kv4AttnArgs& a, const TcShape& s, float* part, float2* ml, void* kept, cudaStream_t st) {
    unsigned char* q = a.mass ? static_cast<unsigned char*>(kept) : nullptr;
    const cudaError_t e = a.c.D == 128 ? (s.nb == 2 ? launch_tc<128, 2>(a, s, part, ml, q, st) : launch_tc<128, 1>(a, s, part, ml, q, st))
                                       : (s.nb == 2 ? launch_tc<64, 2>(a, s, part, ml, q, st) : launch_tc<64, 1>(a, s, part, ml, q, st));
    if (e != cudaSuccess || !a.mass) return e;
    return launch_kv4_mass_tc(a, s, q, st);
}

}  // namespace qw
