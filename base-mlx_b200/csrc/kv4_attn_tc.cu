// Attention over the 4-bit KV cache for many rows per kv head (prompt chunks),
// on the tcgen05 tensor cores.
//
// A thread block takes NB = 1 or 2 blocks of 128 columns (row, query head) of one
// (sequence, kv head) and walks the keys they see in tiles of 64:
//   S_g = Q_g N_g^T   per 64-element group g: Q (fp16, scaled per column as in
//                     kv4_tile.cuh) against the packed integers, which enter as
//                     fp16 subnormals (n 2^-24, the odd nibbles 16 n 2^-24
//                     against q / 16): exact products, fp32 sums in TMEM
//   x = c sum_g s_g S_g + sum_g b_g q_g - m      fp32, one thread per column
//   P = 2^x           fp16 in TMEM, over S_0's columns
//   O += P V          V dequantised to fp16 in shared memory, fp32 sums in TMEM
// V is taken times 2^-E with E the exponent of the block's largest value (found
// first, from scales and biases alone), so any bf16 range fits fp16; the running
// maximum moves only when a score passes it by 2^4 (P <= 2^15), and then O is
// rescaled in TMEM.
//
// Roles: warps 0 .. 4 NB - 1 one column per thread (with NB = 2 one column
// block's softmax overlaps the other's products); four warps copy packed rows
// (cp.async ring) and expand them, once for all column blocks; one lane of the
// last warp issues the products.  Every wait is bounded: a lost arrival sets
// QW_DERR_TIMEOUT and the block still frees its TMEM and ends.
#include "kv4_tc.h"
#include "kv4_tile.cuh"
#include "smem_attr.h"

namespace qw {
namespace {

using namespace kv4;

constexpr int CM = 128;      // columns of a column block
constexpr int KT = 64;       // keys of a tile
constexpr int STAGES = 3;    // packed tiles in flight
constexpr int TABS = 4;      // score tables: a tile's is read until the products of the next tile but one are issued
template <int NB>
constexpr int THREADS = 128 * NB + 160;
constexpr float BASE = 11.f;          // P = 2^(x - max + 11)
constexpr float RAISE = BASE + 4.f;   // a larger exponent raises the maximum
constexpr float UNSET = -3.0e38f;
constexpr unsigned long long TIMEOUT_NS = 2000000000ull;

// Shared memory, from a 1 KB aligned base.
template <int D, int NB>
struct Plan {
    static constexpr int GR = D / 64, OPB = GR * KT * 128;
    static constexpr int Q = 1024;                    // [NB][GR][128 rows][128 B], swizzled
    static constexpr int K = Q + NB * GR * CM * 128;  // [2][GR][64 keys][128 B], swizzled
    static constexpr int V = K + 2 * OPB;             // the same, read along the keys
    static constexpr int TAB = V + 2 * OPB;           // [TABS][K scale, K bias][GR][64] fp32
    static constexpr int PACK = TAB + TABS * 2 * GR * KT * 4;
    static constexpr int PW = KT * D / 2, PS = KT * GR * 2, PACKB = 2 * PW + 4 * PS;
    static constexpr int BYTES = PACK + STAGES * PACKB + 1024;
    // TMEM columns of a column block: S_0, (S_1), O; P over S_0
    static constexpr uint32_t TO = GR * KT, TB = GR * KT + D, TMEM = NB * TB;
};

QW_DEV unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
QW_DEV bool wait_ns(uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const unsigned long long t0 = now_ns();
    while (!mbar_try_wait(bar, parity))
        if (now_ns() - t0 > TIMEOUT_NS) return false;
    return true;
}
QW_DEV void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
QW_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
QW_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
QW_DEV void commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 128-byte-swizzled operand rows of 64 fp16: descriptor version 1, 1 KB between 8-row groups; along_keys:
// the matrix' k runs over the rows and its 64-element blocks lie `lead` bytes apart.
QW_DEV uint64_t desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// kind::f16, fp32 sums, fp16 operands, A along k, B along k or (bit 16) along n; M = 128.
__host__ __device__ constexpr uint32_t idesc(int n, bool b_along_n) {
    return (1u << 4) | (b_along_n ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(CM >> 4) << 24);
}
QW_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}
QW_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}
QW_DEV void ld16(uint32_t addr, float (&v)[16]) {
    uint32_t r[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
QW_DEV void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
QW_DEV void st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
QW_DEV void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
QW_DEV uint32_t h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
QW_DEV __half2 as_h2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
QW_DEV uint32_t as_u(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// 16-byte chunk c of a swizzled operand row.  A word fills one chunk, its elements in the order 0, 4, 1, 5, 2, 6, 3, 7.
QW_DEV uint32_t chunk_at(int row, int c) { return (uint32_t)row * 128 + (uint32_t)((c ^ (row & 7)) << 4); }

QW_DEV unsigned long long pack2(float lo, float hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
QW_DEV void unpack2(unsigned long long v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
QW_DEV unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
QW_DEV unsigned long long mul2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
QW_DEV unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

template <int D, int NB>
__global__ void __launch_bounds__(THREADS<NB>, 1) kv4_attn_tc_kernel(const Kv4AttnArgs a, int ncb, int nsplit, float* part, float2* pml) {
    using P = Plan<D, NB>;
    constexpr int GR = P::GR, CB = CM * NB, PW0 = 4 * NB;  // columns of the block, first producer warp
    extern __shared__ unsigned char tc_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)tc_raw + 1023) & ~(uintptr_t)1023);
    // barriers: tile i uses [i & 1] of the paired ones; those per column block count tiles
    uint64_t* k_full = reinterpret_cast<uint64_t*>(sm);  // K operand and table written
    uint64_t* k_free = k_full + 2;                        // products Q N of every column block done
    uint64_t* v_full = k_free + 2;
    uint64_t* v_free = v_full + 2;
    uint64_t* s_full = v_free + 2;                        // per column block: scores in TMEM
    uint64_t* p_full = s_full + 2;
    uint64_t* pv_done = p_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + 2);
    float* vmax = reinterpret_cast<float*>(tmem_slot + 2);  // [4] producers' warps
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

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
    const int nt = (keys + KT - 1) / KT, t0 = (int)((long long)nt * sp / nsplit), t1 = (int)((long long)nt * (sp + 1) / nsplit);
    const int all = a.causal ? min(T, rw.off + i_first + 1) : T;  // keys that every column sees
    const size_t seg = ((size_t)b * a.c.heads + h) * ncb + cb;

    const int col = min(tid, CB - 1), c = cb * CB + col, i_row = c / G, head = h * G + c % G;
    const bool row = c < C && i_row < rw.n;
    bf16* out = a.out + (b * a.os.b + (long long)i_row * a.os.s + (long long)head * a.os.h);
    const size_t lse_at = ((size_t)b * a.S + i_row) * a.Hq + head;
    if (t0 == t1) {  // nothing to see: zeros (a split's empty share is skipped by the joining kernel)
        if (nsplit == 1 && tid < CB && c < C) {
            for (int d = 0; d < D; d += 8) *reinterpret_cast<uint4*>(out + d) = make_uint4(0u, 0u, 0u, 0u);
            if (a.lse) a.lse[lse_at] = -INFINITY;
        }
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + i, 128);
            mbar_init(k_free + i, 1);
            mbar_init(v_full + i, 128);
            mbar_init(v_free + i, 1);
            mbar_init(s_full + i, 2);
            mbar_init(p_full + i, 128);
            mbar_init(pv_done + i, 1);
        }
        fence_mbar_init();
    }
    if (warp == PW0 + 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(P::TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }

    const Rows rows = head_rows<D>(a.c, (size_t)b * a.c.heads + h);
    const int key_end = min(T, t1 * KT);  // this block's keys end here
    const int pt = tid - CB;              // producer thread
    auto fetch = [&](int i) {  // tile t0 + i into stage i % STAGES, 16-byte pieces; zeros past the last key
        if (t0 + i < t1) {
            const int key0 = (t0 + i) * KT;
            const uint32_t dst = smem_u32(sm + P::PACK + (i % STAGES) * P::PACKB);
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int j = 0; j < P::PW / 16; j += 128) {
                    const int piece = j + pt;
                    const bool ok = key0 + piece / (D / 32) < T;
                    cp_async16_zfill(dst + w * P::PW + piece * 16, ok ? rows.w[w] + (size_t)key0 * (D / 2) + piece * 16 : rows.w[w], ok);
                }
            constexpr int SP = P::PS / 16, KPP = KT / SP;  // pieces of a scale array, keys of a piece
            if (pt < 4 * SP) {
                const int arr = pt / SP, piece = pt % SP;
                const unsigned char* base = arr & 2 ? (arr & 1 ? rows.b[1] : rows.s[1]) : (arr & 1 ? rows.b[0] : rows.s[0]);
                const bool ok = key0 + piece * KPP < T;
                cp_async16_zfill(dst + 2 * P::PW + pt * 16, ok ? base + (size_t)key0 * (2 * GR) + piece * 16 : base, ok);
            }
        }
        cp_async_commit();
    };

    float cc = 0.f, q0 = 0.f, q1 = 0.f;  // the column's score constants (softmax threads)
    if (warp < PW0) {
        // Q operand: column `col`, elements of a chunk in the order of an expanded word
        const bf16* src = a.q + (b * a.qs.b + (long long)i_row * a.qs.s + (long long)head * a.qs.h);
        float mx = 0.f, sum[GR];
#pragma unroll
        for (int g = 0; g < GR; ++g) {
            sum[g] = 0.f;
            if (row)
#pragma unroll 4
                for (int k = 0; k < 8; ++k) {
                    const uint4 u = *reinterpret_cast<const uint4*>(src + 64 * g + 8 * k);
                    const uint32_t X[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float lo = bits_lo_f(X[e]), hi = bits_hi_f(X[e]);
                        sum[g] += lo + hi;
                        mx = fmaxf(mx, fmaxf(fabsf(lo), fabsf(hi)));
                    }
                }
        }
        const int ex = max((int)(__float_as_uint(mx) >> 23) - 127, -100);
        const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
        cc = ldexpf(a.scale * LOG2E, ex - 14 + 24);
        q0 = sum[0] * (a.scale * LOG2E);
        q1 = sum[GR - 1] * (a.scale * LOG2E);
#pragma unroll
        for (int g = 0; g < GR; ++g)
#pragma unroll 4
            for (int k = 0; k < 8; ++k) {
                uint4 u = make_uint4(0u, 0u, 0u, 0u);
                if (row) u = *reinterpret_cast<const uint4*>(src + 64 * g + 8 * k);
                const uint32_t X[4] = {u.x, u.y, u.z, u.w};
                float x[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[2 * e] = bits_lo_f(X[e]) * up;
                    x[2 * e + 1] = bits_hi_f(X[e]) * up;
                }
                *reinterpret_cast<uint4*>(sm + P::Q + ((col >> 7) * GR + g) * CM * 128 + chunk_at(col & 127, k)) =
                    make_uint4(h2(x[0], x[4]), h2(x[1] * 0.0625f, x[5] * 0.0625f), h2(x[2], x[6]), h2(x[3] * 0.0625f, x[7] * 0.0625f));
            }
        fence_proxy_async_smem();
    } else if (warp < PW0 + 4) {
#pragma unroll
        for (int i = 0; i < STAGES - 1; ++i) fetch(i);
        // largest |value| that the block's V rows can stand for: max(|b|, |b + 15 s|) (a NaN counts as nothing here)
        float mx = 0.f;
        const uint32_t* s = reinterpret_cast<const uint32_t*>(rows.s[1]);
        const uint32_t* z = reinterpret_cast<const uint32_t*>(rows.b[1]);
        constexpr int KW = 2 / GR;  // keys of a 32-bit word of scales (rows end at a multiple of 16)
#pragma unroll 8
        for (int w = t0 * KT / KW + pt; w < (key_end + KW - 1) / KW; w += 128) {
            const uint32_t us = s[w], uz = z[w];
            const float z0 = bits_lo_f(uz), z1 = bits_hi_f(uz);
            float m = fmaxf(fabsf(z0), fabsf(fmaf(15.f, bits_lo_f(us), z0)));
            if (GR == 2 || w * KW + 1 < key_end) m = fmaxf(m, fmaxf(fabsf(z1), fabsf(fmaf(15.f, bits_hi_f(us), z1))));
            mx = fmaxf(mx, m);
        }
        mx = warp_max(mx);
        if (lane == 0) vmax[warp - PW0] = mx;
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    // V enters as value 2^(13 - ev): below 2^14
    const float vm = fmaxf(fmaxf(vmax[0], vmax[1]), fmaxf(vmax[2], vmax[3]));
    const int ev = max((int)(__float_as_uint(fminf(vm, 3.0e38f)) >> 23) - 127, -100);
    const int n_tiles = t1 - t0;
    bool ok = true;

    if (warp < PW0) {
        // ---- softmax: one column per thread ------------------------------------------------------
        const int blk = warp >> 2;
        const uint32_t tm = tmem + blk * P::TB + ((uint32_t)(32 * (warp & 3)) << 16);
        const int vis = row ? (a.causal ? min(T, rw.off + i_row + 1) : T) : 0;
        const unsigned long long c2 = pack2(cc, cc), q02 = pack2(q0, q0), q12 = pack2(q1, q1);
        float nm = 0.f, l = 0.f, thr = UNSET;  // BASE - maximum; up to thr the maximum stays
        for (int i = 0; i < n_tiles; ++i) {
            const int key0 = (t0 + i) * KT;
            if (ok && !wait_ns(s_full + blk, i & 1)) ok = false;
            fence_after();
            const float* tab = reinterpret_cast<const float*>(sm + P::TAB) + (i % TABS) * 2 * GR * KT;
            const unsigned long long nm2 = pack2(nm, nm);
            float x[KT];
#pragma unroll
            for (int k = 0; k < KT; k += 16) {
                float a0[16], a1[16];
                ld16(tm + k, a0);
                if (GR == 2) ld16(tm + KT + k, a1);
                wait_ld();
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const ulonglong2 s0 = *reinterpret_cast<const ulonglong2*>(tab + k + e),
                                     z0 = *reinterpret_cast<const ulonglong2*>(tab + GR * KT + k + e);
                    unsigned long long d[2] = {mul2(s0.x, pack2(a0[e], a0[e + 1])), mul2(s0.y, pack2(a0[e + 2], a0[e + 3]))};
                    unsigned long long u[2] = {fma2(z0.x, q02, nm2), fma2(z0.y, q02, nm2)};
                    if (GR == 2) {
                        const ulonglong2 s1 = *reinterpret_cast<const ulonglong2*>(tab + KT + k + e),
                                         z1 = *reinterpret_cast<const ulonglong2*>(tab + 3 * KT + k + e);
                        d[0] = fma2(s1.x, pack2(a1[e], a1[e + 1]), d[0]);
                        d[1] = fma2(s1.y, pack2(a1[e + 2], a1[e + 3]), d[1]);
                        u[0] = fma2(z1.x, q12, u[0]);
                        u[1] = fma2(z1.y, q12, u[1]);
                    }
                    unpack2(fma2(c2, d[0], u[0]), x[k + e], x[k + e + 1]);
                    unpack2(fma2(c2, d[1], u[1]), x[k + e + 2], x[k + e + 3]);
                }
            }
            if (key0 + KT > all)
#pragma unroll
                for (int k = 0; k < KT; ++k)
                    if (key0 + k >= vis) x[k] = -INFINITY;
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < KT; ++k) top = fmaxf(top, x[k]);
            if (__any_sync(0xffffffffu, top > thr)) {
                // raise the maximum of the columns that ask for it, and rescale what they have summed
                float al = 1.f;
                if (top > thr) {
                    const float up = BASE - top;
                    al = thr == UNSET ? 0.f : ex2(up);  // the column's first key: nothing summed so far
                    nm += up;
                    thr = RAISE;
#pragma unroll
                    for (int k = 0; k < KT; ++k) x[k] += up;
                }
                if (i > 0) {  // P V of the tile before is complete: the products of this one came after it
#pragma unroll 1
                    for (int d = 0; d < D; d += 16) {
                        float o[16];
                        uint32_t r[16];
                        ld16(tm + P::TO + d, o);
                        wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(o[e] * al);
                        st16(tm + P::TO + d, r);
                    }
                    l *= al;
                }
            }
            unsigned long long l2[2] = {0ull, 0ull};
#pragma unroll
            for (int k = 0; k < KT; k += 32) {
                uint32_t r[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float p0 = ex2(x[k + 2 * e]), p1 = ex2(x[k + 2 * e + 1]);
                    l2[e & 1] = add2(l2[e & 1], pack2(p0, p1));
                    r[e] = h2(p0, p1);
                }
                st16(tm + k / 2, r);
            }
            float l0, l1;
            unpack2(add2(l2[0], l2[1]), l0, l1);
            l += l0 + l1;
            wait_st();
            fence_before();
            arrive(p_full + blk);
        }
        if (ok && !wait_ns(pv_done + blk, (n_tiles - 1) & 1)) ok = false;
        fence_after();
        // ---- output ---------------------------------------------------------------------------------
        const bool has = row && l != 0.f;
        const float f = nsplit == 1 ? (has ? 1.f / l : 0.f) : 1.f;
        const float e0 = __uint_as_float((uint32_t)(127 - 13) << 23), e1 = __uint_as_float((uint32_t)(127 + ev) << 23);
        const size_t slot = (seg * nsplit + sp) * CB + col;
#pragma unroll 1
        for (int d = 0; d < D; d += 16) {
            float o[16];
            ld16(tm + P::TO + d, o);
            wait_ld();
#pragma unroll
            for (int g = 0; g < 16; g += 8) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = o[g + (e < 4 ? 2 * e : 2 * e - 7)] * f * e0 * e1;  // columns hold 0, 4, 1, 5, ...
                if (!ok || c >= C) continue;
                if (nsplit == 1) {
                    *reinterpret_cast<uint4*>(out + d + g) =
                        has ? make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]))
                            : make_uint4(0u, 0u, 0u, 0u);
                } else {
                    float* dst = part + slot * D + d + g;
                    *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
        }
        if (ok && c < C) {
            if (nsplit == 1) {
                if (a.lse) a.lse[lse_at] = has ? (log2f(l) - nm) * LN2 : -INFINITY;
            } else {
                pml[slot] = make_float2(l != 0.f ? -nm : M0, l);
            }
        }
    } else if (warp < PW0 + 4) {
        // ---- producers: packed rows -> operands ----------------------------------------------------
        const int key = pt & 63, g = D == 128 ? pt >> 6 : 0, half = D == 128 ? 0 : pt >> 6;  // D = 64: half a row each
        constexpr int WPT = D == 128 ? 8 : 4;  // words per thread
        const __half2 k1024 = __float2half2_rn(1024.f);
        const float dn = __uint_as_float((uint32_t)(127 + 13 - max(ev, -100)) << 23);
        for (int i = 0; i < n_tiles; ++i) {
            cp_async_wait<STAGES - 2>();
            asm volatile("bar.sync 1, 128;" ::: "memory");  // every producer's pieces have landed, and all have left the stage to be refilled
            fetch(i + STAGES - 1);
            const unsigned char* pk = sm + P::PACK + (i % STAGES) * P::PACKB;
            const int kpos = (t0 + i) * KT + key;
            const bool valid = kpos < T;  // rows past the last key may hold anything in their scales
            uint32_t w[WPT];
            {
                const uint4* p = reinterpret_cast<const uint4*>(pk + key * (D / 2) + g * 32 + half * 16);
#pragma unroll
                for (int j = 0; j < WPT / 4; ++j) {
                    const uint4 u = p[j];
                    w[4 * j] = u.x;
                    w[4 * j + 1] = u.y;
                    w[4 * j + 2] = u.z;
                    w[4 * j + 3] = u.w;
                }
            }
            const uint16_t* sc = reinterpret_cast<const uint16_t*>(pk + 2 * P::PW) + key * GR + g;
            float ks = valid ? u16_to_f(sc[0]) : 0.f, kz = valid ? u16_to_f(sc[P::PS / 2]) : 0.f;
            float vs = valid ? u16_to_f(sc[P::PS]) : 0.f, vz = valid ? u16_to_f(sc[3 * P::PS / 2]) : 0.f;
            if (!(fabsf(vs) < INFINITY) || !(fabsf(vz) < INFINITY)) {
                // a NaN in V reaches the rows that see the key through its score, and no other row
                kz = vs + vz + INFINITY - INFINITY;
                vs = vz = 0.f;
            }
            if (ok && i > 1 && !wait_ns(k_free + (i & 1), ((i - 2) >> 1) & 1)) ok = false;
            unsigned char* kd = sm + P::K + (i & 1) * P::OPB + g * KT * 128;
#pragma unroll
            for (int j = 0; j < WPT; ++j)
                *reinterpret_cast<uint4*>(kd + chunk_at(key, half * 4 + j)) =
                    make_uint4(nib_even(w[j]), nib_odd(w[j]), nib_even(w[j] >> 8), nib_odd(w[j] >> 8));
            if (half == 0) {
                float* tab = reinterpret_cast<float*>(sm + P::TAB) + (i % TABS) * 2 * GR * KT + g * KT + key;
                tab[0] = ks;
                tab[GR * KT] = kz;
            }
            fence_proxy_async_smem();
            arrive(k_full + (i & 1));
            {
                const uint4* p = reinterpret_cast<const uint4*>(pk + P::PW + key * (D / 2) + g * 32 + half * 16);
#pragma unroll
                for (int j = 0; j < WPT / 4; ++j) {
                    const uint4 u = p[j];
                    w[4 * j] = u.x;
                    w[4 * j + 1] = u.y;
                    w[4 * j + 2] = u.z;
                    w[4 * j + 3] = u.w;
                }
            }
            const __half2 s2 = __float2half2_rn(vs * dn), z2 = __float2half2_rn(vz * dn);
            if (ok && i > 1 && !wait_ns(v_free + (i & 1), ((i - 2) >> 1) & 1)) ok = false;
            unsigned char* vd = sm + P::V + (i & 1) * P::OPB + g * KT * 128;
#pragma unroll
            for (int j = 0; j < WPT; ++j) {
                uint32_t o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    o[e] = as_u(__hfma2(__hsub2(as_h2(((w[j] >> (4 * e)) & 0x000F000Fu) | 0x64006400u), k1024), s2, z2));
                *reinterpret_cast<uint4*>(vd + chunk_at(key, half * 4 + j)) = make_uint4(o[0], o[1], o[2], o[3]);
            }
            fence_proxy_async_smem();
            arrive(v_full + (i & 1));
        }
        cp_async_wait<0>();
    } else if (lane == 0) {
        // ---- products ------------------------------------------------------------------------------------
        const uint32_t qb = smem_u32(sm + P::Q), kb = smem_u32(sm + P::K), vb = smem_u32(sm + P::V);
        auto scores = [&](int blk, int i) {  // S of tile i; the arrival passes on what the producers wrote
#pragma unroll
            for (int g = 0; g < GR; ++g)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    mma_ss(tmem + blk * P::TB + g * KT, desc(qb + (blk * GR + g) * CM * 128 + 32 * k, 16),
                           desc(kb + (i & 1) * P::OPB + g * KT * 128 + 32 * k, 16), idesc(KT, false), k != 0 ? 1u : 0u);
            commit(s_full + blk);
            arrive(s_full + blk);
            if (blk == NB - 1) commit(k_free + (i & 1));
        };
        if (!wait_ns(k_full, 0)) ok = false;
        if (ok) {
            fence_after();
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) scores(blk, 0);
        }
        for (int i = 0; i < n_tiles && ok; ++i) {
            if (!wait_ns(v_full + (i & 1), (i >> 1) & 1)) ok = false;
#pragma unroll
            for (int blk = 0; blk < NB; ++blk) {
                if (ok && !wait_ns(p_full + blk, i & 1)) ok = false;
                if (!ok) break;
                fence_after();
#pragma unroll
                for (int k = 0; k < KT / 16; ++k)
                    mma_ts(tmem + blk * P::TB + P::TO, tmem + blk * P::TB + 8 * k, desc(vb + (i & 1) * P::OPB + 16 * 128 * k, KT * 128),
                           idesc(D, true), (i | k) != 0 ? 1u : 0u);
                commit(pv_done + blk);
                if (blk == NB - 1) commit(v_free + (i & 1));
                if (i + 1 < n_tiles) {  // S_0 holds P until its product is done
                    if ((blk == 0 && !wait_ns(k_full + ((i + 1) & 1), ((i + 1) >> 1) & 1)) || !wait_ns(pv_done + blk, i & 1)) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    scores(blk, i + 1);
                }
            }
        }
    }
    if (!ok && a.err) atomicOr(a.err, (int)QW_DERR_TIMEOUT);
    fence_before();
    __syncthreads();
    if (warp == PW0 + 4) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(P::TMEM) : "memory");
    }
}

// Joins the splits' partials.  One block per (column, sequence), one thread per dimension.
template <int D>
__global__ void __launch_bounds__(D) kv4_attn_tc_join_kernel(const Kv4AttnArgs a, int cb_size, int ncb, int nsplit, const float* part, const float2* pml) {
    const int b = blockIdx.y, G = a.Hq / a.c.heads, d = threadIdx.x, h = blockIdx.x % a.Hq, i = blockIdx.x / a.Hq;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, nullptr, false);
    const int c = i * G + h % G, cb = c / cb_size, C = G * a.S;
    const int i_last = min(rw.n, (min(C, (cb + 1) * cb_size) - 1) / G + 1) - 1;
    const int T = rw.off + rw.n, nt = ((a.causal ? min(T, rw.off + i_last + 1) : T) + KT - 1) / KT;
    bf16* dst = a.out + (b * a.os.b + (long long)i * a.os.s + (long long)h * a.os.h) + d;
    float* lse = a.lse ? a.lse + ((size_t)b * a.S + i) * a.Hq + h : nullptr;
    pdl_wait();
    float M = M0, o = 0.f, l = 0.f;
    if (i < rw.n) {
        const size_t s0 = ((((size_t)b * a.c.heads + h / G) * ncb + cb) * nsplit) * cb_size + c % cb_size;
        for (int s = 0; s < nsplit; ++s)
            if ((long long)nt * s / nsplit != (long long)nt * (s + 1) / nsplit) M = fmaxf(M, pml[s0 + (size_t)s * cb_size].x);
        for (int s = 0; s < nsplit; ++s)
            if ((long long)nt * s / nsplit != (long long)nt * (s + 1) / nsplit) {
                const float2 ml = pml[s0 + (size_t)s * cb_size];
                const float f = half_pow(ml.x - M);
                l = fmaf(ml.y * f, f, l);
                o = fmaf(part[(s0 + (size_t)s * cb_size) * D + d] * f, f, o);
            }
    }
    *dst = f2bf(l != 0.f ? o / l : 0.f);
    if (lse && d == 0) *lse = l != 0.f ? (M + log2f(l)) * LN2 : -INFINITY;
}

template <typename K, typename... Args>
cudaError_t launch(K kernel, dim3 grid, dim3 block, size_t smem, cudaStream_t st, bool pdl, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int D, int NB>
cudaError_t launch_tc(const Kv4AttnArgs& a, const TcShape& sp, float* part, float2* ml, cudaStream_t st) {
    constexpr int smem = Plan<D, NB>::BYTES;
    cudaError_t e = ensure_max_dyn_smem(kv4_attn_tc_kernel<D, NB>, smem);
    if (e != cudaSuccess) return e;
    const long long blocks = (long long)sp.ncb * sp.nsplit * a.c.heads * a.c.batch;
    if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
    e = launch(kv4_attn_tc_kernel<D, NB>, dim3((unsigned)blocks), dim3(THREADS<NB>), smem, st, false, a, sp.ncb, sp.nsplit, part, ml);
    if (e != cudaSuccess || sp.nsplit == 1) return e;
    return launch(kv4_attn_tc_join_kernel<D>, dim3((unsigned)(a.S * a.Hq), a.c.batch), dim3(D), 0, st, true, a, CM * NB, sp.ncb,
                  sp.nsplit, (const float*)part, (const float2*)ml);
}

}  // namespace

TcShape kv4_tc_shape(const Kv4View& c, int S, int Hq, int num_sms) {
    const long long C = (long long)(Hq / c.heads) * S;
    TcShape s;
    s.nb = C > CM ? 2 : 1;
    s.ncb = (int)((C + CM * s.nb - 1) / (CM * s.nb));
    // splits of the keys: fill rounds of one block per SM, at least four tiles each if the cache were
    // full; a split costs a partial's write and read, counted as a tenth of a round
    const long long segs = (long long)s.ncb * c.heads * c.batch;
    s.nsplit = 1;
    float best = 1e30f;
    for (int n = 1; n <= 64 && (n == 1 || n * 4 * KT <= c.max_pos); ++n) {
        const float t = (float)((segs * n + num_sms - 1) / num_sms) / n * (1.f + 0.1f * (n - 1));
        if (t < best) {
            best = t;
            s.nsplit = n;
        }
    }
    s.part_rows = s.nsplit > 1 ? (size_t)segs * s.nsplit * CM * s.nb : 0;
    return s;
}

cudaError_t launch_kv4_attn_tc(const Kv4AttnArgs& a, const TcShape& s, float* part, float2* ml, cudaStream_t st) {
    if (a.c.D == 128) return s.nb == 2 ? launch_tc<128, 2>(a, s, part, ml, st) : launch_tc<128, 1>(a, s, part, ml, st);
    return s.nb == 2 ? launch_tc<64, 2>(a, s, part, ml, st) : launch_tc<64, 1>(a, s, part, ml, st);
}

}  // namespace qw
