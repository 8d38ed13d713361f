// Attention weights of the 4-bit KV cache for many rows per kv head, on the
// tcgen05 tensor cores:
//   mass[key] += sum over the columns (row, query head) that see it of 2^(c S - log2-sum-exp),
//   S = K' Q^T + C* Q*^T, the operands of kv4_attn_tc.cu with keys along M.
//
// With a key per TMEM lane the sum over the columns is a thread's own, in a
// fixed order, and needs neither atomics nor exchanges.  A thread block keeps two
// tiles of 128 keys expanded in shared memory and walks the columns, 128 at a
// time: the Q operand that the attention kernel built and kept arrives by one
// bulk copy (one tile of keys per block instead would read 36 KB of Q from L2 per
// 128 x 128 scores, more than L2 gives).  A thread takes one key of either tile
// and a quarter of the columns, so that a column's factor and log-sum-exp, read
// from shared memory, serve two scores (serving one, those reads were the bound:
// a broadcast of 16 bytes takes four of the 128-byte cycles); S is double buffered
// in TMEM, Q three times in shared memory.  What bounds it is 2^x (16 a clock and
// SM) next to shared memory: a tile of columns takes 3000 cycles, 2050 of them the
// powers.  512 rows of 16 heads on 8 kv heads, 4096 keys: 20 us (with scores by
// mma.sync and queries unpacked per block: 63 us).
#include "kv4_launch.h"
#include "kv4_tc.h"
#include "kv4_tcgen.cuh"
#include "smem_attr.h"

namespace qw {
namespace {

using namespace kv4;

constexpr int KBLOCKS = 2;                    // key tiles of a thread block
constexpr int PW = 16;                        // the product warp; the others: a quarter of the columns per 4 warps
constexpr int MTHREADS = 32 * PW + 32;
constexpr int QSTAGES = 3;
// Column tables.  A thread arrives on s_free for tile i while it still reads table i, so that arrival only tells that it has
// left table i - 1; table i + 2 is written behind the arrivals for tile i - 2 and must lie on table i - 3 or an older one.
constexpr int TABLES = 8;
static_assert(TABLES >= 5 && (TABLES & (TABLES - 1)) == 0, "tables i - 2 to i + 2 are in use at a time");
constexpr uint32_t MASS_TMEM = 2 * KBLOCKS * CM;

// Shared memory, from a 1 KB aligned base: barriers, column tables, sums, K operands, Q operands.
template <int D>
struct MassPlan {
    static constexpr int GR = D / 64;
    static constexpr int KB = GR * KT * 128 + KT * 32, QB = q_block_bytes(D);
    static constexpr int TAB = 1024;                   // [TABLES][64 column pairs]{factor x 2, -log2-sum-exp x 2}
    static constexpr int SUM = TAB + TABLES * CM * 8;       // [column quarter][key tile][key]
    static constexpr int K = SUM + 4 * KBLOCKS * KT * 4;   // [key tile]{[GR][128 keys][128 B] swizzled; C*}
    static constexpr int Q = K + KBLOCKS * KB;
    static constexpr int BYTES = Q + QSTAGES * QB + 1024;
    static_assert(K % 1024 == 0 && KB % 1024 == 0 && QB % 1024 == 0, "swizzled rows start at a multiple of 1 KB");
};

template <int D>
__global__ void __launch_bounds__(MTHREADS, 1) kv4_mass_tc_kernel(const Kv4AttnArgs a, int blocks, const unsigned char* kept) {
    using P = MassPlan<D>;
    constexpr int GR = P::GR;
    extern __shared__ unsigned char mass_raw[];
    unsigned char* sm = reinterpret_cast<unsigned char*>(((uintptr_t)mass_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* q_full = reinterpret_cast<uint64_t*>(sm);  // [QSTAGES] Q operand arrived
    uint64_t* s_full = q_full + QSTAGES;                 // [2] scores in TMEM
    uint64_t* s_free = s_full + 2;                       // [2] scores read, and the table two tiles on written
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(s_free + 2);
    float* kmax = reinterpret_cast<float*>(tmem_slot + 2);  // [8]
    float* tab = reinterpret_cast<float*>(sm + P::TAB);
    float* sums = reinterpret_cast<float*>(sm + P::SUM);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = blockIdx.y, b = blockIdx.z, G = a.Hq / a.c.heads;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, nullptr, false);
    const int T = rw.off + rw.n, key0 = blockIdx.x * KBLOCKS * KT;
    const int c_end = rw.n * G;
    if (key0 >= T || c_end == 0) {
        pdl_wait();
        return;
    }
    // columns that see none of the block's keys come first when causal
    const int c_first = a.causal ? max(0, key0 - rw.off) * G / CM * CM : 0;
    const int n_tiles = (c_end - c_first + CM - 1) / CM;
    if (tid == 0) {
        for (int i = 0; i < QSTAGES; ++i) mbar_init(q_full + i, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full + i, 1);
            mbar_init(s_free + i, 32 * PW);
        }
        fence_mbar_init();
    }

    // ---- K operands (the cache is older than the kernel before this one) ------------------------------------
    const Rows rows = head_rows<D>(a.c, (size_t)b * a.c.heads + h);
    uint32_t cs = 0, cz = 0;
    if (warp < KBLOCKS * KT / 32) {
        if (key0 + tid < T) {
            cs = group_pair<GR>(rows.s[0], key0 + tid);
            cz = group_pair<GR>(rows.b[0], key0 + tid);
        }
        const float m = warp_max(fmaxf(reach(bits_lo_f(cs), bits_lo_f(cz)), reach(bits_hi_f(cs), bits_hi_f(cz))));
        if (lane == 0) kmax[warp] = m;
    }
    __syncthreads();
    float m = 0.f;
#pragma unroll
    for (int w = 0; w < KBLOCKS * KT / 32; ++w) m = fmaxf(m, kmax[w]);
    const int ek = top_exponent(m);
    const float kup = __uint_as_float((uint32_t)(127 + 7 - ek) << 23);
    if (warp < PW) {
        constexpr int CPR = D / 32, PER = KT * CPR / 256;
        const int kb = warp >> 3, k0 = key0 + kb * KT;
        const uint4* src = reinterpret_cast<const uint4*>(rows.w[0]) + (size_t)k0 * CPR;
        const uint16_t* s = reinterpret_cast<const uint16_t*>(rows.s[0]) + (size_t)k0 * GR;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int p = (tid & 255) + 256 * j, key = p / CPR;
            const bool in = k0 + key < T;
            const uint4 w = in ? src[p] : make_uint4(0u, 0u, 0u, 0u);
            expand_piece<D>(w, p, sm + P::K + kb * P::KB, Centred(in ? u16_to_f(s[key * GR + ((p % CPR) >> 1)]) * kup : 0.f));
        }
        if (tid < KBLOCKS * KT)
            store_offsets<GR>(sm + P::K + tid / KT * P::KB + GR * KT * 128, tid % KT, cs, cz, kup);
    }

    pdl_wait();  // the rows' log-sum-exp and the Q operands are the attention kernels'
    if (warp == PW) {  // (only now: a kernel that this one waits for may still want its TMEM)
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(MASS_TMEM)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // the next tile's Q operand (product warp)
    int issued = 0;
    auto load = [&](size_t image) {
        if (issued >= n_tiles) return;
        if (lane == 0) {
            mbar_arrive_expect_tx(q_full + issued % QSTAGES, P::QB);
            bulk_g2s(sm + P::Q + issued % QSTAGES * P::QB, kept + (image + issued) * P::QB, P::QB, q_full + issued % QSTAGES);
        }
        ++issued;
    };
    const size_t image = ((size_t)b * a.c.heads + h) * blocks + c_first / CM;
    if (warp == PW)
        for (int i = 0; i < QSTAGES; ++i) load(image);
    const float* factor = reinterpret_cast<const float*>(kept + (size_t)a.c.batch * a.c.heads * blocks * P::QB) + image * CM;
    // threads 0 .. 127: factor and log-sum-exp of a column (2^-inf where there is none)
    auto fetch = [&](int i) {
        const int c = c_first + i * CM + tid;
        if (tid >= CM || c >= c_end) return make_float2(0.f, INFINITY);
        return make_float2(factor[i * CM + tid], a.lse[((size_t)b * a.S + c / G) * a.Hq + h * G + c % G]);
    };
    auto put = [&](int i, float2 v) {
        if (tid >= CM) return;
        float* t = tab + (i & (TABLES - 1)) * 2 * CM + (tid >> 1) * 4 + (tid & 1);
        t[0] = ldexpf(v.x, ek - 7);
        t[2] = -v.y * LOG2E;
    };
    const float2 v0 = fetch(0), v1 = fetch(1);
    float2 ahead = fetch(2);
    put(0, v0);
    put(1, v1);
    fence_proxy_async_smem();
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    bool ok = true;

    if (warp < PW) {
        const int quarter = warp >> 2, row = 32 * (warp & 3) + lane;
        const uint32_t tm = tmem + quarter * 32 + ((uint32_t)(32 * (warp & 3)) << 16);
        // first column that sees a key: the thread's two, the block's first, its last
        auto first_of = [&](int k) { return a.causal ? max(0, k - rw.off) * G : 0; };
        int mine[KBLOCKS];
#pragma unroll
        for (int n = 0; n < KBLOCKS; ++n) mine[n] = first_of(key0 + n * KT + row) - c_first - quarter * 32;
        const int c_all = first_of(key0 + KBLOCKS * KT - 1);
        float total[KBLOCKS] = {0.f, 0.f};
        for (int i = 0; i < n_tiles; ++i) {
            const int buf = i & 1;
            if (ok && i > 1 && !wait_bar(s_free + buf, ((i - 2) >> 1) & 1)) ok = false;
            if (ok && !wait_bar(s_full + buf, (i >> 1) & 1)) ok = false;
            fence_after();
            put(i + 2, ahead);  // over the table of tile i + 2 - TABLES, which every thread has left
            ahead = fetch(i + 3);
            unsigned long long s2[KBLOCKS] = {0ull, 0ull};
#pragma unroll 1
            for (int r = 0; r < 32; r += 16) {  // 16 columns of both tiles at a time: 32 would spill
                float x[KBLOCKS][16];
#pragma unroll
                for (int n = 0; n < KBLOCKS; ++n) ld16(tm + (buf * KBLOCKS + n) * CM + r, x[n]);
                wait_ld();
                if (r == 16) {
                    fence_before();
                    arrive(s_free + buf);
                }
                const ulonglong2* t = reinterpret_cast<const ulonglong2*>(tab + (i & (TABLES - 1)) * 2 * CM) + quarter * 16 + r / 2;
                if (c_first + i * CM >= c_all) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const ulonglong2 f = t[e];
#pragma unroll
                        for (int n = 0; n < KBLOCKS; ++n) {
                            float p0, p1;
                            unpack2(fma2(pack2(x[n][2 * e], x[n][2 * e + 1]), f.x, f.y), p0, p1);
                            s2[n] = add2(s2[n], pack2(ex2(p0), ex2(p1)));
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const ulonglong2 f = t[e];
#pragma unroll
                        for (int n = 0; n < KBLOCKS; ++n) {
                            const int from = mine[n] - i * CM - r;
                            float p0, p1;
                            unpack2(fma2(pack2(x[n][2 * e], x[n][2 * e + 1]), f.x, f.y), p0, p1);
                            s2[n] = add2(s2[n], pack2(2 * e < from ? 0.f : ex2(p0), 2 * e + 1 < from ? 0.f : ex2(p1)));
                        }
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < KBLOCKS; ++n) {
                float s0, s1;
                unpack2(s2[n], s0, s1);
                total[n] += s0 + s1;
            }
        }
#pragma unroll
        for (int n = 0; n < KBLOCKS; ++n) sums[(quarter * KBLOCKS + n) * KT + row] = total[n];
        asm volatile("bar.sync 1, %0;" ::"n"(32 * PW) : "memory");
        if (tid < KBLOCKS * KT && key0 + tid < T && ok) {
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < 4; ++w) sum += sums[w * KBLOCKS * KT + tid];
            a.mass[((size_t)b * a.c.heads + h) * a.c.max_pos + key0 + tid] += sum;
        }
    } else {
        const uint32_t qa = smem_u32(sm + P::Q), ka = smem_u32(sm + P::K);
        const uint64_t qd = desc(qa, 16), kd = desc(ka, 16), qx = desc16(qa + GR * CM * 128), kx = desc16(ka + GR * KT * 128);
        auto at = [](uint64_t d, uint32_t bytes) { return d + (bytes >> 4); };
        int i = 0;
        for (; i < n_tiles; ++i) {
            const int buf = i & 1;
            if (!wait_bar(q_full + i % QSTAGES, (i / QSTAGES) & 1)) ok = false;
            if (ok && i > 1 && !wait_bar(s_free + buf, ((i - 2) >> 1) & 1)) ok = false;
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            fence_after();
            const uint32_t qo = i % QSTAGES * P::QB;
#pragma unroll
            for (int n = 0; n < KBLOCKS; ++n) {
                const uint32_t d = tmem + (buf * KBLOCKS + n) * CM, ko = n * P::KB;
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_ss(d, at(kd, ko + (k >> 2) * KT * 128 + 32 * (k & 3)), at(qd, qo + (k >> 2) * CM * 128 + 32 * (k & 3)), idesc(CM, false),
                           k != 0 ? 1u : 0u);
                mma_ss(d, at(kx, ko), at(qx, qo), idesc(CM, false), 1u);
            }
            commit(s_full + buf);
            if (i > 0 && issued < n_tiles) {  // the stage of tile i - 1 is free once its products are done
                if (!wait_bar(s_full + (buf ^ 1), ((i - 1) >> 1) & 1)) ok = false;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                load(image);
            }
        }
        for (; !ok && i < issued; ++i) wait_bar(q_full + i % QSTAGES, (i / QSTAGES) & 1);  // copies still on their way
    }
    if (!ok && a.err) atomicOr(a.err, (int)QW_DERR_TIMEOUT);
    fence_before();
    __syncthreads();
    if (warp == PW) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(MASS_TMEM) : "memory");
    }
}

template <int D>
cudaError_t launch_mass(const Kv4AttnArgs& a, const TcShape& s, const unsigned char* kept, cudaStream_t st) {
    constexpr int smem = MassPlan<D>::BYTES;
    const cudaError_t e = ensure_max_dyn_smem(kv4_mass_tc_kernel<D>, smem);
    if (e != cudaSuccess) return e;
    const dim3 grid((a.c.max_pos + KBLOCKS * KT - 1) / (KBLOCKS * KT), a.c.heads, a.c.batch);
    return launch(kv4_mass_tc_kernel<D>, grid, dim3(MTHREADS), smem, 1, st, a, s.ncb * s.nb, kept);
}

}  // namespace

cudaError_t launch_kv4_mass_tc(const Kv4AttnArgs& a, const TcShape& s, const unsigned char* kept, cudaStream_t st) {
    return a.c.D == 128 ? launch_mass<128>(a, s, kept, st) : launch_mass<64>(a, s, kept, st);
}

}  // namespace qw
