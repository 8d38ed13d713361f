// Attention arithmetic on 32-key tiles of a 4-bit KV cache, shared by the
// attention and the weight-accumulation kernels.
//
// A warp multiplies a tile's packed rows without dequantising them.  With
// n the stored integers, group g of a key row stands for s_g n + b_g, so
//   <q, k_j>       = sum_g s_jg <q_g, n_jg> + b_jg sum(q_g)
//   sum_j p_j v_j  = sum_j (p_j s_jg) n_jg + sum_j p_j b_jg
// and the tensor cores (mma m16n8k16, fp16 operands, fp32 sums) only see n and
// q or n and p s.  A nibble left in the low bits of an fp16 is the subnormal
// n 2^-24 (16 n 2^-24 for the odd ones): four ANDs and a shift unpack a word,
// and the products are exact.  Keys (for the scores) and dimensions (for the
// values) are the M index, 8 query columns per kv head the N index, so the few
// rows of a decode step waste little of the tensor cores.
//
// Operand rounding:
//   * q: bf16 times a power of two per column (largest magnitude at 2^14) is
//     exact in fp16; elements 2^25 below the largest lose bits that are below
//     2^-39 of it.
//   * p s: fp16 (relative 2^-11; normal numbers down to 2^-25 of the largest
//     p s) -- taken times a power of two that keeps the largest near 2^11, see
//     State.  The output is bf16, whose own half step is eight times that.
// Everything else (scores, maxima, sums, the bias part of the output) is fp32.
#pragma once
#include <cuda_fp16.h>

#include "kv4.h"

namespace qw {
namespace kv4 {

constexpr int TK = 32;            // keys of a tile
constexpr float M0 = -3.0e38f;    // base exponent of a column before its first key
constexpr float LAZY = 4.f;       // the maximum is raised when a score passes it by 2^LAZY
constexpr int LOG2_PSCALE = 11;   // p s / sref <= 2^LAZY enters fp16 times 2^11: at most 2^15
constexpr float LN2 = 0.6931471805599453f, LOG2E = 1.4426950408889634f;

// Shared memory of a tile: K words, V words (16-byte chunks at chunk_pos), then
// scales and biases of K and of V.
template <int D>
struct Tile {
    static constexpr int GR = D / 64, ROWB = D / 2, CPR = D / 32;  // groups, word bytes and 16-byte chunks of a row
    static constexpr int VW = TK * ROWB, SB = 2 * TK * ROWB, SBB = TK * GR * 2;
    static constexpr int BYTES = SB + 4 * SBB;
    // Chunk c of key k: eight consecutive keys' chunks c, the rows of an ldmatrix, lie in eight bank groups.
    static QW_DEV int chunk_pos(int k, int c) {
        return D == 128 ? 4 * k + (c ^ ((k >> 1) & 3)) : 2 * k + (c ^ ((k >> 2) & 1));
    }
};

QW_DEV void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
QW_DEV void cp_async16_zfill(uint32_t dst, const void* src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

// Global pointers of one (sequence, kv head).
struct Rows {
    const unsigned char* w[2];
    const unsigned char *s[2], *b[2];
};
template <int D>
QW_DEV Rows head_rows(const Kv4View& c, size_t bh) {
    Rows r;
    const size_t row = bh * c.max_pos;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        r.w[i] = reinterpret_cast<const unsigned char*>(c.p[i].w) + row * (D / 2);
        r.s[i] = reinterpret_cast<const unsigned char*>(c.p[i].s) + row * (D / 32);
        r.b[i] = reinterpret_cast<const unsigned char*>(c.p[i].b) + row * (D / 32);
    }
    return r;
}

// Copies tiles of 32 keys, key0, key0 + 32 step, ... into shared memory, by the
// lanes of one warp; rows from T on arrive as zeros (scales and biases in pieces
// of 16 bytes, so up to 7 rows past T may hold what the cache has there).  The
// addresses only move by constants from tile to tile.
template <int D>
struct TileLoader {
    using L = Tile<D>;
    static constexpr int CH = TK * L::CPR;                 // 16-byte chunks of the tile's words
    static constexpr int SC = L::SBB / 16, KPC = TK / SC;  // 16-byte pieces of a scale array, keys of a piece
    const unsigned char *w0, *w1, *sb;                     // this lane's first chunk of K and V words, its scale piece
    const unsigned char* safe;                             // a readable address for chunks that are not copied
    int key, keys;                                         // first key of the next tile, keys from tile to tile
    QW_DEV void start(const Rows& r, int key0, int step, int lane) {
        const int arr = (lane / SC) & 3, piece = lane % SC;
        key = key0;
        keys = step * TK;
        safe = r.w[0];
        w0 = r.w[0] + (size_t)key0 * L::ROWB + lane * 16;
        w1 = r.w[1] + (size_t)key0 * L::ROWB + lane * 16;
        sb = (arr & 2 ? (arr & 1 ? r.b[1] : r.s[1]) : (arr & 1 ? r.b[0] : r.s[0])) + (size_t)key0 * (2 * L::GR) + piece * 16;
    }
    // into the tile at shared address `dst`, of which `to` is this lane's first chunk of words
    QW_DEV void copy(uint32_t dst, uint32_t to, int T, int lane) {
        const uint32_t sd = dst + L::SB + lane * 16;
        if (key + TK <= T) {
            // a row group of 32 chunks further on is a fixed distance away on both sides
#pragma unroll
            for (int i = 0; i < CH / 32; ++i) {
                cp_async16(to + i * 512, w0 + i * 512);
                cp_async16(to + L::VW + i * 512, w1 + i * 512);
            }
            if (lane < 4 * SC) cp_async16(sd, sb);
        } else {
#pragma unroll
            for (int i = 0; i < CH / 32; ++i) {
                const bool ok = key + (lane + 32 * i) / L::CPR < T;
                cp_async16_zfill(to + i * 512, ok ? w0 + i * 512 : safe, ok);
                cp_async16_zfill(to + L::VW + i * 512, ok ? w1 + i * 512 : safe, ok);
            }
            if (lane < 4 * SC) {
                const bool ok = key + lane % SC * KPC < T;
                cp_async16_zfill(sd, ok ? sb : safe, ok);
            }
        }
        key += keys;
        w0 += (size_t)keys * L::ROWB;
        w1 += (size_t)keys * L::ROWB;
        sb += (size_t)keys * (2 * L::GR);
    }
};

// Query columns of a warp: 8 NT of them.
template <int D, int NT>
struct Cols {
    static constexpr int GR = D / 64;
    uint32_t f[GR][4][NT][2];                 // B fragments: column lane / 4; [2 j + half] of word 4 j + lane % 4
    float c[NT][2];                           // columns 2 (lane % 4) + {0, 1}: score = c sum_g s_g <n_g, f_g> + sum_g b_g q_g
    uint32_t qb[NT];                          // the q_g as a B operand of three bf16 terms (24 bits): k = 2 term + group
};

// A lane's part of column lane / 4: words t and t + 4 of every group (t = lane % 4); null: zeros.
template <int D>
struct RawCol {
    uint4 u[D / 64][2];
};
template <int D>
QW_DEV void fetch_col(RawCol<D>& o, const bf16* src, int lane) {
    const int t = lane & 3;
#pragma unroll
    for (int g = 0; g < D / 64; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j)
            o.u[g][j] = src ? *reinterpret_cast<const uint4*>(src + 64 * g + 32 * j + 8 * t) : make_uint4(0u, 0u, 0u, 0u);
}
// Column lane / 4 of n-tile n from its bf16 row; scale * log2(e) goes into c and q.
template <int D, int NT>
QW_DEV void load_cols(Cols<D, NT>& o, int n, const RawCol<D>& raw, float scale, int lane) {
    constexpr int GR = D / 64;
    const int t = lane & 3;
    float x[GR][16], sum[GR], mx = 0.f;
#pragma unroll
    for (int g = 0; g < GR; ++g) {
        sum[g] = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t X[4] = {raw.u[g][j].x, raw.u[g][j].y, raw.u[g][j].z, raw.u[g][j].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[g][8 * j + 2 * e] = bits_lo_f(X[e]);
                x[g][8 * j + 2 * e + 1] = bits_hi_f(X[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            sum[g] += x[g][e];
            mx = fmaxf(mx, fabsf(x[g][e]));
        }
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // 2^ex is the largest magnitude's power of two; columns below 2^-100 keep that scaling
    const int ex = max((int)(__float_as_uint(mx) >> 23) - 127, -100);
    const float up = __uint_as_float((uint32_t)(127 + 14 - ex) << 23);
    const float down = ldexpf(scale * LOG2E, ex - 14 + 24);
#pragma unroll
    for (int g = 0; g < GR; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                // k-steps of word j: nibbles (0, 4) and 16 x (1, 5), then (2, 6) and 16 x (3, 7)
                const float* v = &x[g][8 * j + 2 * s];
                const __half2 lo = __floats2half2_rn(v[0] * up, v[4] * up);
                const __half2 hi = __floats2half2_rn(v[1] * up * 0.0625f, v[5] * up * 0.0625f);
                o.f[g][2 * j + s][n][0] = *reinterpret_cast<const uint32_t*>(&lo);
                o.f[g][2 * j + s][n][1] = *reinterpret_cast<const uint32_t*>(&hi);
            }
#pragma unroll
    for (int e = 0; e < 2; ++e) o.c[n][e] = __shfl_sync(0xffffffffu, down, 8 * t + 4 * e);  // a lane of column 2 t + e
    uint32_t qb = 0;
#pragma unroll
    for (int g = 0; g < GR; ++g) {
        const float v = sum[g] * (scale * LOG2E), hi = bfr(v), mid = bfr(v - hi), lo = v - hi - mid;
        qb |= (uint32_t)f_to_bf16bits(t == 0 ? hi : t == 1 ? mid : t == 2 ? lo : 0.f) << (16 * g);
    }
    o.qb[n] = qb;
}

// D[16x8] (fp32) = A[16x8] (bf16) * B[8x8] (bf16) + C: a0 row g, a1 row g + 8, b column g, k = 2 t + {0, 1}.
QW_DEV void mma_bf16_k8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b, const float (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%8,%9,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(b), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Four 8 x 8 matrices of 16-bit halves; lane l gives the row address of matrix l / 8, row l % 8.
QW_DEV void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
QW_DEV void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// K operand of one 16-key block: rows g and g + 8 (g = lane / 4), words 4 j + t of every group.
template <int D>
struct KeyBlock {
    uint32_t w[D / 64][2][2];  // [group][row half][j]
};
template <int D>
QW_DEV void read_keys(KeyBlock<D>& o, uint32_t tile, int kb, int lane) {
    using L = Tile<D>;
    uint32_t r[4];
    if (D == 128) {  // a matrix = 8 keys x chunk (one word of each per lane); chunk = 2 group + j
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            ldmatrix4(r, tile + L::chunk_pos(lane & 7, lane >> 3) * 16 + (16 * kb + 8 * h) * L::ROWB);
#pragma unroll
            for (int c = 0; c < 4; ++c) o.w[(c >> 1) % L::GR][h][c & 1] = r[c];
        }
    } else {  // matrices: keys 0-7 chunks 0, 1, keys 8-15 chunks 0, 1
        ldmatrix4(r, tile + L::chunk_pos((lane & 7) + 8 * (lane >> 4), (lane >> 3) & 1) * 16 + 16 * kb * L::ROWB);
#pragma unroll
        for (int c = 0; c < 4; ++c) o.w[0][c >> 1][c & 1] = r[c];
    }
}
// acc[group][n][4] = integer dot products of the block's keys with the columns
template <int D, int NT>
QW_DEV void key_dots(float (&acc)[D / 64][NT][4], const KeyBlock<D>& k, const Cols<D, NT>& c) {
#pragma unroll
    for (int gr = 0; gr < D / 64; ++gr) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[gr][n][e] = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t a = k.w[gr][0][j] >> (8 * s), b = k.w[gr][1][j] >> (8 * s);
                const uint32_t a0 = nib_even(a), a1 = nib_even(b), a2 = nib_odd(a), a3 = nib_odd(b);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    mma_f16(acc[gr][n], a0, a1, a2, a3, c.f[gr][2 * j + s][n][0], c.f[gr][2 * j + s][n][1], acc[gr][n]);
            }
    }
}

// The bf16 of every group of key k, packed; array 0 K scales, 1 K biases, 2 V scales, 3 V biases.
template <int D>
QW_DEV uint32_t read_packed(const unsigned char* tile, int arr, int k) {
    using L = Tile<D>;
    const unsigned char* p = tile + L::SB + arr * L::SBB + k * (2 * L::GR);
    return D == 128 ? *reinterpret_cast<const uint32_t*>(p) : (uint32_t)*reinterpret_cast<const uint16_t*>(p);
}
template <int GR>
QW_DEV void unpack(uint32_t u, float (&v)[GR]) {
    v[0] = bits_lo_f(u);
    if (GR == 2) v[GR - 1] = bits_hi_f(u);
}

QW_DEV float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// 2^(d / 2), applied twice where a base changes by d: bases may lie more than 2^126 apart
QW_DEV float half_pow(float d) { return ex2(0.5f * d); }
QW_DEV uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Running softmax and output of a warp's columns.  Lane (g, t) holds the
// columns 2 t + {0, 1} of every n-tile; l and bs are the lane's share (its
// keys).  o, l and bs are relative to 2^-nm = 2^m sref / PSCALE with m the
// column's running maximum and sref a power of two above the largest value
// scale met so far, so exp2(x + nm) s <= 2^LAZY PSCALE enters fp16, and above 2^-60 of
// the largest bias: p b <= 2^(LAZY + 71) keeps the bias sums in range where every scale is 0.
// (p ends at 2^-126, which is 2^-136 s of the largest p: 2^-36 at a scale s of 2^100.  Taking scales
// and biases times a power of two from there on was measured: 1 to 4 % of every decode.)
template <int D, int NT>
struct State {
    static constexpr int GR = D / 64;
    // [4 group + i]: rows g -> dimension 64 group + 32 (i / 2) + 4 g + 2 (i % 2), rows g + 8 -> the next (times 16)
    float o[D / 16][NT][4];
    float nm[NT][4];         // {column 0, 1, 0, 1}: the C operand of a score tile; 0 before the first key
    float thr[NT][2];        // largest exponent that leaves the base as it is; M0 before the first key
    float l[NT][2], bs[GR][NT][2];
    float sref;
    QW_DEV void init() {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                nm[n][e] = nm[n][2 + e] = 0.f;
                thr[n][e] = M0;
                l[n][e] = 0.f;
#pragma unroll
                for (int g = 0; g < GR; ++g) bs[g][n][e] = 0.f;
            }
        set_sref(0.f);
    }
    // sref: the power of two above s, at least 2^-79
    QW_DEV void set_sref(float s) {
        const uint32_t e = min(max(__float_as_uint(s) >> 23, 47u) + 1u, 254u);
        sref = __uint_as_float(e << 23);
    }
    QW_DEV float shift() const { return (float)(LOG2_PSCALE + 127 - (int)(__float_as_uint(sref) >> 23)); }  // log2(PSCALE / sref)
    // the base exponent of column (n, e), M0 before the first key
    QW_DEV float base(int n, int e) const { return thr[n][e] == M0 ? M0 : -nm[n][e]; }
};

// One tile: keys [key0, key0 + 32) of which vis[n][e] (absolute) are visible to
// column (n, e).  EDGE: some key of the tile is not visible to some column.
// WEIGHTS: the scores (base 2, -inf for hidden keys) go to scores[key - key0][column], rows of cp columns.
template <int D, int NT, bool EDGE, bool WEIGHTS>
QW_DEV void attend_tile(State<D, NT>& st, const Cols<D, NT>& cols, const unsigned char* tile, int key0, int T,
                        const int (&vis)[NT][2], int lane, float* scores, int cp) {
    const uint32_t tile_s = smem_u32(tile);
    using L = Tile<D>;
    constexpr int GR = L::GR;
    const int g = lane >> 2;
    float acc[2][GR][NT][4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
        KeyBlock<D> k;
        read_keys<D>(k, tile_s, kb, lane);
        key_dots<D, NT>(acc[kb], k, cols);
    }
    float ks[4][GR];
    uint32_t kz[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        unpack<GR>(read_packed<D>(tile, 0, 8 * r + g), ks[r]);
        kz[r] = read_packed<D>(tile, 1, 8 * r + g);
    }
    // x[kb][n][2 r + e]: score of key 16 kb + 8 r + g and column 2 t + e, less the column's base
    float x[2][NT][4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            mma_bf16_k8(x[kb][n], kz[2 * kb], kz[2 * kb + 1], cols.qb[n], st.nm[n]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 2 * kb + (e >> 1);
                float d = ks[r][0] * acc[kb][0][n][e];
                if (GR == 2) d = fmaf(ks[r][GR - 1], acc[kb][GR - 1][n][e], d);
                x[kb][n][e] = fmaf(cols.c[n][e & 1], d, x[kb][n][e]);
                if (EDGE && key0 + 8 * r + g >= vis[n][e & 1]) x[kb][n][e] = -INFINITY;
            }
        }
    // largest value scale of the tile, or 2^-60 of its largest bias (lane = key)
    float vs[4][GR], vz[4][GR], smax;
    unpack<GR>(read_packed<D>(tile, 2, lane), vs[0]);
    unpack<GR>(read_packed<D>(tile, 3, lane), vz[0]);
    smax = fmaxf(fabsf(vs[0][0]), fabsf(vz[0][0]) * 0x1p-60f);
    if (GR == 2) smax = fmaxf(fmaxf(smax, fabsf(vs[0][GR - 1])), fabsf(vz[0][GR - 1]) * 0x1p-60f);
    if (EDGE && key0 + lane >= T) smax = 0.f;
    if (!(smax < 2.0e37f)) smax = 0.f;  // past the range times 15: must not push the values of other rows to zero
    bool raise = smax > st.sref;
    float top[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            top[n][e] = fmaxf(fmaxf(x[0][n][e], x[0][n][2 + e]), fmaxf(x[1][n][e], x[1][n][2 + e]));
            raise = raise || top[n][e] > st.thr[n][e];
        }
    if (__any_sync(0xffffffffu, raise)) {
        // rare: raise the column maxima to the tile's, the scale reference to its largest scale
        const float before = st.shift();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) smax = fmaxf(smax, __shfl_xor_sync(0xffffffffu, smax, o));
        if (smax > st.sref) st.set_sref(smax);
        const float now = st.shift();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float mx = top[n][e];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const bool seen = st.thr[n][e] != M0;
                if (seen) mx = fmaxf(mx, before);        // the old maximum's exponent
                if (!seen && mx == -INFINITY) continue;  // still no key for this column
                const float by = now - mx, al = seen ? half_pow(by) : 0.f;
                st.nm[n][e] += by;
                st.nm[n][2 + e] += by;
                st.thr[n][e] = now + LAZY;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    x[kb][n][e] += by;
                    x[kb][n][2 + e] += by;
                }
                st.l[n][e] = st.l[n][e] * al * al;
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) st.bs[gr][n][e] = st.bs[gr][n][e] * al * al;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    st.o[i][n][e] = st.o[i][n][e] * al * al;
                    st.o[i][n][2 + e] = st.o[i][n][2 + e] * al * al;
                }
            }
    }
    if (WEIGHTS) {
        float* row = scores + g * cp + 2 * (lane & 3);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int n = 0; n < NT; ++n)
                if (8 * n + 2 * (lane & 3) < cp && (!EDGE || key0 + 8 * r + g < T))
                    *reinterpret_cast<float2*>(row + 8 * r * cp + 8 * n) =
                        make_float2(x[r >> 1][n][2 * (r & 1)] - st.nm[n][0], x[r >> 1][n][2 * (r & 1) + 1] - st.nm[n][1]);
    }
    // probabilities, their sums, and p s in the B-operand layout (keys along k)
    uint32_t pb[2][GR][NT][2];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        unpack<GR>(read_packed<D>(tile, 2, 8 * r + g), vs[r]);
        unpack<GR>(read_packed<D>(tile, 3, 8 * r + g), vz[r]);
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float x0 = x[kb][n][2 * r], x1 = x[kb][n][2 * r + 1];
                const float p0 = ex2(x0), p1 = ex2(x1);
                const int kr = 2 * kb + r;
                st.l[n][0] += p0;
                st.l[n][1] += p1;
#pragma unroll
                for (int gr = 0; gr < GR; ++gr) {
                    float a0 = p0 * vs[kr][gr], a1 = p1 * vs[kr][gr];
                    if (EDGE) {  // a hidden key's scale and bias may be anything
                        a0 = x0 == -INFINITY ? 0.f : a0;
                        a1 = x1 == -INFINITY ? 0.f : a1;
                        st.bs[gr][n][0] = x0 == -INFINITY ? st.bs[gr][n][0] : fmaf(p0, vz[kr][gr], st.bs[gr][n][0]);
                        st.bs[gr][n][1] = x1 == -INFINITY ? st.bs[gr][n][1] : fmaf(p1, vz[kr][gr], st.bs[gr][n][1]);
                    } else {
                        st.bs[gr][n][0] = fmaf(p0, vz[kr][gr], st.bs[gr][n][0]);
                        st.bs[gr][n][1] = fmaf(p1, vz[kr][gr], st.bs[gr][n][1]);
                    }
                    const __half2 h = __floats2half2_rn(a0, a1);
                    pb[kb][gr][n][r] = transpose8x8(*reinterpret_cast<const uint32_t*>(&h));
                }
            }
    // Transposed 8 x 8 matrices of the packed rows put halfword h of two neighbouring keys, four
    // dimensions each, into one register: h = 8 m + g, dimensions 4 h + {0, 1, 2, 3}.
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) {
            uint32_t w[4];  // [m & 1][keys 0-7, 8-15 of the block]
            ldmatrix4_trans(w, tile_s + L::VW + L::chunk_pos((lane & 7) + (lane & 8), 2 * gr + (lane >> 4)) * 16 + 16 * kb * L::ROWB);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t u = w[2 * (i >> 1)] >> (8 * (i & 1)), v = w[2 * (i >> 1) + 1] >> (8 * (i & 1));
                const uint32_t a0 = nib_even(u), a1 = nib_odd(u), a2 = nib_even(v), a3 = nib_odd(v);
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    mma_f16(st.o[4 * gr + i][n], a0, a1, a2, a3, pb[kb][gr][n][0], pb[kb][gr][n][1], st.o[4 * gr + i][n]);
            }
        }
}

// The state's share of the output (times the sum's base), dimensions 64 gr + 32 (i / 2) + 4 g +
// 2 (i % 2) + {0, 1} of columns 2 t + e: what the tensor cores summed plus the bias sums (lanes reduced before).
template <int D, int NT>
QW_DEV float2 out_pair(const State<D, NT>& st, int gr, int i, int n, int e) {
    return make_float2(fmaf(st.o[4 * gr + i][n][e], QW_NIB_SCALE, st.bs[gr][n][e]),
                       fmaf(st.o[4 * gr + i][n][2 + e], QW_NIB_SCALE_ODD, st.bs[gr][n][e]));
}
// Sums over the lanes of a column (its keys).
template <int D, int NT>
QW_DEV void reduce_lanes(State<D, NT>& st) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                st.l[n][e] += __shfl_xor_sync(0xffffffffu, st.l[n][e], o);
#pragma unroll
                for (int gr = 0; gr < D / 64; ++gr) st.bs[gr][n][e] += __shfl_xor_sync(0xffffffffu, st.bs[gr][n][e], o);
            }
}

}  // namespace kv4
}  // namespace qw
