// What the tcgen05 kernels of the 4-bit cache attention share: operand layouts,
// descriptors, TMEM access, packed arithmetic.
#pragma once
#include "kv4_tile.cuh"

namespace qw {
namespace kv4 {

constexpr int CM = 128;  // columns (row, query head) of a column block
constexpr int KT = 128;  // keys of a tile

// Operand rows of 128 columns: [D / 64][128 rows][128 B] fp16, swizzled; then the 16-wide extra step.
__host__ __device__ constexpr int q_block_bytes(int D) { return D / 64 * CM * 128 + CM * 32; }

// Bounded wait: every poll suspends for a while, 2^22 of them are far beyond any tile's time.
QW_DEV bool wait_bar(uint64_t* bar, uint32_t parity) { return mbar_wait_bounded(bar, parity); }
QW_DEV void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
QW_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
QW_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The product warp runs as a whole, so that its control flow and descriptors stay in uniform
// registers; one elected lane issues.
QW_DEV void commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar))
        : "memory");
}
// 128-byte-swizzled operand rows of 64 fp16: descriptor version 1, 1 KB between 8-row groups; along_keys:
// the matrix' k runs over the rows and its 64-element blocks lie `lead` bytes apart.
QW_DEV uint64_t desc(uint32_t addr, uint32_t lead) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) |
           (2ull << 61);
}
// The 16-wide extra operand: 8 rows x 16 bytes make a block of 128 bytes, [row / 8][k / 8][row % 8][16 B], no swizzle.
QW_DEV uint64_t desc16(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(128u >> 4) << 16) | ((uint64_t)(256u >> 4) << 32) | (1ull << 46);
}
QW_DEV uint32_t at16(int row, int khalf) { return (uint32_t)(row >> 3) * 256 + khalf * 128 + (row & 7) * 16; }
// kind::f16, fp32 sums, fp16 operands, A along k, B along k or (bit 16) along n; M = 128.
__host__ __device__ constexpr uint32_t idesc(int n, bool b_along_n) {
    return (1u << 4) | (b_along_n ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(CM >> 4) << 24);
}
QW_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}
QW_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(accumulate)
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
QW_DEV unsigned long long add2(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Piece p (words 4 (p % CPR) .. of key p / CPR) of a tile's packed rows to the swizzled operand rows at dst, each
// word's nibble pairs through `value`, which gets (n_j, n_{j + 4}) at bits 6 .. 9 of its halves: n 2^-18 as fp16.  With two groups the second one's words go out
// in another order (e ^ 2): the eight lanes of a store phase (two keys, all pieces) hit eight different chunk columns.
template <int D, typename F>
QW_DEV void expand_piece(const uint4& w, int p, unsigned char* dst, F&& value) {
    constexpr int CPR = D / 32;
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    const int key = p / CPR, q = p % CPR, g = q >> 1;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t v = g ? u[e ^ 2] : u[e];
        uint32_t o[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) o[n] = value((n < 2 ? v << (6 - 4 * n) : v >> (4 * n - 6)) & 0x03C003C0u);
        *reinterpret_cast<uint4*>(dst + g * KT * 128 + chunk_at(key, 4 * (q & 1) + (g ? e ^ 2 : e))) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}
// K' of a pair: s (n - 8) = (16 + n) s - 24 s in one exact step (24 s has 10 bits).
struct Centred {
    __half2 s2, m24;
    QW_DEV explicit Centred(float s) : s2(__float2half2_rn(s)), m24(__hmul2(s2, __float2half2_rn(-24.f))) {}
    QW_DEV uint32_t operator()(uint32_t n) const { return as_u(__hfma2(as_h2(n | 0x4C004C00u), s2, m24)); }
};
// C* of one key (`scale`, `bias`: its groups' bf16 pairs): 2^6 c kup in two fp16 terms, k = 5 g + {0..4}: hi, lo, hi, lo, hi.
template <int GR>
QW_DEV void store_offsets(unsigned char* dst, int row, uint32_t scale, uint32_t bias, float kup) {
    __half c[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) c[e] = __float2half_rn(0.f);
#pragma unroll
    for (int g = 0; g < GR; ++g) {
        const float x = fmaf(8.f, g ? bits_hi_f(scale) : bits_lo_f(scale), g ? bits_hi_f(bias) : bits_lo_f(bias)) * kup * 64.f;
        const __half hi = __float2half_rn(x), lo = __float2half_rn(x - __half2float(hi));
        c[5 * g] = c[5 * g + 2] = c[5 * g + 4] = hi;
        c[5 * g + 1] = c[5 * g + 3] = lo;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        uint32_t r[4];
#pragma unroll
        for (int f = 0; f < 4; ++f) r[f] = as_u(__halves2half2(c[8 * e + 2 * f], c[8 * e + 2 * f + 1]));
        *reinterpret_cast<uint4*>(dst + at16(row, e)) = make_uint4(r[0], r[1], r[2], r[3]);
    }
}
// The largest magnitude that a group's scale and bias can stand for; one that is not finite counts as nothing, so that
// it does not push the other keys' values to zero.
QW_DEV bool finite(float s, float z) { return 0.25f * fabsf(z) + 0.25f * fabsf(fmaf(15.f, s, z)) < INFINITY; }
QW_DEV float reach(float s, float z) { return finite(s, z) ? fmaxf(fabsf(z), fabsf(fmaf(15.f, s, z))) : 0.f; }
// The exponent of a largest magnitude m: K enters times 2^(7 - ek), V times 2^(-2 - ev).
QW_DEV int top_exponent(float m) { return max((int)(__float_as_uint(m) >> 23) - 127, -100); }
// The bf16 of every group of a key.
template <int GR>
QW_DEV uint32_t group_pair(const unsigned char* base, size_t key) {
    return GR == 2 ? *reinterpret_cast<const uint32_t*>(base + key * 4) : (uint32_t)*reinterpret_cast<const uint16_t*>(base + key * 2);
}

}  // namespace kv4
}  // namespace qw
