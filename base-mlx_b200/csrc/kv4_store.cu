// Writing rows into the 4-bit KV cache and reading them back.
//
// Quantisation of a group x[0..63] of a bf16 row (the format of the model
// weights): bias = min x, scale = bf16((max x - min x) / 15),
// q = clamp(round_half_even((x - bias) / scale), 0, 15), q = 0 where scale = 0.
// A group that holds a NaN or an infinity gets scale = bias = NaN, so all of
// it reads back as NaN.
//
// Every q is the rounding of the exact quotient, ties to even.  Ties are common
// (about one element in 500: x, bias and scale are 8-bit numbers), so they are
// settled without a branch, from the exact remainder.
#include "kv4.h"

namespace qw {
namespace {

constexpr int NT = 256;
// threads of one row: 8 values each (one packed word)
template <int D>
constexpr int TPR = D / 8;

QW_DEV float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// bf16((hi - lo) / 15) of the exact difference, rounded through fp32
QW_DEV float group_scale(float hi, float lo) {
    const float d = __fsub_rn(hi, lo);
    float s = __fmul_rn(d, 1.0f / 15.0f);
    // next to a midpoint of two bf16 values, past the fp32 range or below bf16's normal numbers the
    // fp32 steps (off by less than 3 units) may decide wrongly
    const uint32_t low = __float_as_uint(s) & 0xFFFFu;
    if (!(d <= 3.0e38f) || (low >= 0x7FF8u && low <= 0x8008u) || s < 1.2e-38f)
        s = __double2float_rn(((double)hi - (double)lo) / 15.0);
    return bfr(s);
}

// Word of the eight values' clamp(round_half_even((x - bias) / scale), 0, 15).
// quantize8_any decides every element in fp64; quantize8 gives the same word
// in fp32 where every x - bias is exact in it.
//
// x - bias may take more than fp64's 53 bits: it is d + e with d the fp64 difference
// and e its rounding error (Knuth's two-sum).  Halves (n + 1/2) scale have 13 bits, so d's
// neighbours among the fp64 numbers include them: a d that is not a half is farther from the
// next one than e, its quotient does not round to one, and e decides only where d is a half.
__device__ __noinline__ uint32_t quantize8_any(uint4 u, float bias, float scale) {
    const uint32_t X[4] = {u.x, u.y, u.z, u.w};
    uint32_t word = 0;
    for (int j = 0; j < 8; ++j) {
        const double x = j & 1 ? bits_hi_f(X[j >> 1]) : bits_lo_f(X[j >> 1]), b = -(double)bias, s = scale;
        const double d = __dadd_rn(x, b);
        double r = rint(d / s);
        const double rem = fma(-r, s, d);  // exact
        if (fabs(rem) == 0.5 * s) {
            const double bv = __dadd_rn(d, -x), e = __dadd_rn(__dadd_rn(x, -__dadd_rn(d, -bv)), __dadd_rn(b, -bv));
            if (rem * e > 0.0) r += rem > 0.0 ? 1.0 : -1.0;  // the quotient lies past the half that d fell on
        }
        word |= (uint32_t)fmin(fmax(r, 0.0), 15.0) << (4 * j);
    }
    return word;
}
QW_DEV uint32_t quantize8(const float (&x)[8], float bias, float scale) {
    // 1.5 2^23 + t rounds t (within 4e-6 of the quotient) to an integer r, the nearest or, next to a
    // half, its neighbour; r is in the low bits of 0x4B400000 + r.  The remainder (x - bias) - r scale
    // is exact, so comparing it with scale / 2 (as bit patterns; a tie counts against an odd r) tells
    // whether r has to move towards it.  A scale that is a normal bf16 is within 2^-9 of
    // (max - min) / 15: 0 <= t < 15.1, and r needs no clamp.
    constexpr float MAGIC = 12582912.f;
    float inv;
    asm("rcp.approx.f32 %0, %1;" : "=f"(inv) : "f"(scale));
    const int half = __float_as_int(0.5f * scale);
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float d = __fsub_rn(x[j], bias), m = __fadd_rn(__fmul_rn(d, inv), MAGIC);
        const int rem = __float_as_int(fmaf(-__fsub_rn(m, MAGIC), scale, d));
        int r = __float_as_int(m);
        if ((rem & 0x7FFFFFFF) + (r & 1) > half) r += (rem >> 31) | 1;
        word += (uint32_t)r << (4 * j);
    }
    return word - 0x4B400000u * 0x11111111u;
}

// Block = one (sequence, K or V, head) and R * NT / TPR consecutive new rows,
// each thread one word of R of them.  Every input is loaded before the first
// is used and before the lengths arrive: the blocks are short, and the latency of
// the loads counts more than their bytes.  4099 rows of 8 heads: 12.7 us (21.5 MB), issue
// slots taken to 71 % and integer units to 64 % by the exact rounding; a warp with an element
// 2^16 below its group's width takes fp64 quotients (18.8 us with 1 % zeros among the keys).
// One row of 8 sequences with its read 3.8 us, latency alone.
template <int D, bool VEC, int R>
__global__ void __launch_bounds__(NT) kv4_append_kernel(const Kv4StoreArgs a) {
    constexpr int T = TPR<D>, RB = NT / T;
    pdl_wait();
    pdl_launch_dependents();
    const int which = blockIdx.y / a.c.heads, h = blockIdx.y % a.c.heads, b = blockIdx.z;
    const int i0 = blockIdx.x * (R * RB) + threadIdx.x / T, e = threadIdx.x % T;
    const bf16* src = a.x[which] + (b * a.xs[which].b + h * a.xs[which].h) + e * 8;
    uint4 u[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = i0 + r * RB;
        u[r] = make_uint4(0u, 0u, 0u, 0u);
        if (i < a.S) {
            const bf16* p = src + i * a.xs[which].s;
            if (VEC) {
                u[r] = __ldcs(reinterpret_cast<const uint4*>(p));
            } else {
                const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
                u[r] = make_uint4(q[0] | ((uint32_t)q[1] << 16), q[2] | ((uint32_t)q[3] << 16),
                                  q[4] | ((uint32_t)q[5] << 16), q[6] | ((uint32_t)q[7] << 16));
            }
        }
    }
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, a.err,
                                blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0);
    const Kv4Part& p = a.c.p[which];
    const size_t row0 = ((size_t)b * a.c.heads + h) * a.c.max_pos + (size_t)rw.off;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint32_t X[4] = {u[r].x, u[r].y, u[r].z, u[r].w};
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = bits_lo_f(X[j]);
            x[2 * j + 1] = bits_hi_f(X[j]);
        }
        float hi = x[0], lo = x[0];
#pragma unroll
        for (int j = 1; j < 8; ++j) {
            hi = max_nan(hi, x[j]);
            lo = fminf(lo, x[j]);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        }
        const int i = i0 + r * RB;
        if (i >= rw.n) continue;
        const bool bad = !(hi <= 3.4e38f) || !(lo >= -3.4e38f);
        float scale = 0.f;
        uint32_t word = 0;
        if (!bad) {
            scale = group_scale(hi, lo);
            if (scale != 0.f) {
                // x - lo is exact in fp32 when no magnitude lies 2^16 below the width (or is 0: also exact,
                // but not worth telling apart); the rest, subnormal scales and widths past the fp32 range go the long way
                float least = lo == 0.f ? INFINITY : fabsf(lo);
#pragma unroll
                for (int j = 0; j < 8; ++j) least = fminf(least, fabsf(x[j]));
                const float width = hi - lo;
                const bool exact = width <= 3.0e38f && least * 65536.f >= width && scale >= 1.2e-38f;
                word = exact ? quantize8(x, lo, scale) : quantize8_any(u[r], lo, scale);
            }
        }
        const size_t row = row0 + i;
        p.w[row * T + e] = word;
        if (e % 8 == 0) {
            reinterpret_cast<uint16_t*>(p.s)[row * (D / 64) + e / 8] = bad ? (uint16_t)0x7FC0 : f_to_bf16bits(scale);
            reinterpret_cast<uint16_t*>(p.b)[row * (D / 64) + e / 8] = bad ? (uint16_t)0x7FC0 : f_to_bf16bits(lo);
        }
    }
}

// The same split for reading back.
template <int D, int R>
__global__ void __launch_bounds__(NT) kv4_read_kernel(const Kv4ReadArgs a) {
    constexpr int T = TPR<D>, RB = NT / T;
    pdl_wait();
    pdl_launch_dependents();
    const int which = blockIdx.y / a.c.heads, h = blockIdx.y % a.c.heads, b = blockIdx.z;
    const int i0 = blockIdx.x * (R * RB) + threadIdx.x / T, e = threadIdx.x % T;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, a.err,
                                blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0);
    if (a.y[which] == nullptr) return;
    const Kv4Part& p = a.c.p[which];
    const size_t row0 = ((size_t)b * a.c.heads + h) * a.c.max_pos + (size_t)rw.off;
    uint32_t w[R];
    float s[R], z[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = i0 + r * RB;
        w[r] = 0u;
        s[r] = z[r] = 0.f;
        if (i < rw.n) {
            const size_t row = row0 + i;
            w[r] = p.w[row * T + e];
            s[r] = bf2f(p.s[row * (D / 64) + e / 8]);
            z[r] = bf2f(p.b[row * (D / 64) + e / 8]);
        }
    }
    bf16* dst = a.y[which] + ((size_t)b * a.S * a.c.heads + h) * D + e * 8;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = i0 + r * RB;
        if (i >= a.S) continue;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)  // 2^23 + q, less 2^23
            v[j] = fmaf(s[r], __fsub_rn(__uint_as_float(0x4B000000u | ((w[r] >> (4 * j)) & 15u)), 8388608.f), z[r]);
        __stcs(reinterpret_cast<uint4*>(dst + (size_t)i * a.c.heads * D),
               make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])));
    }
}

// Rows of a thread: four once one each would make more than two rounds of
// blocks on the GPU (8 of these blocks fit an SM).
int rows_per_thread(const Kv4View& c, int S) {
    const int rb = NT / (c.D / 8);
    return (long long)((S + rb - 1) / rb) * 2 * c.heads * c.batch > 2 * 8 * 148 ? 4 : 1;
}

// Programmatic launch, as the library's other kernels: the blocks start while the kernel before drains and wait
// for it before they touch memory.
template <typename K, typename A>
cudaError_t launch(K kernel, dim3 grid, cudaStream_t st, const A& a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(NT);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <int D, int R>
cudaError_t append_t(const Kv4StoreArgs& a, bool vec, cudaStream_t st) {
    const int rows = R * NT / TPR<D>;
    const dim3 grid((a.S + rows - 1) / rows, 2 * a.c.heads, a.c.batch);
    return vec ? launch(kv4_append_kernel<D, true, R>, grid, st, a) : launch(kv4_append_kernel<D, false, R>, grid, st, a);
}
template <int D, int R>
cudaError_t read_t(const Kv4ReadArgs& a, cudaStream_t st) {
    const int rows = R * NT / TPR<D>;
    const dim3 grid((a.S + rows - 1) / rows, 2 * a.c.heads, a.c.batch);
    return launch(kv4_read_kernel<D, R>, grid, st, a);
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4StoreArgs& a, cudaStream_t st) {
    bool vec = true;
    for (int w = 0; w < 2; ++w)
        vec = vec && (uintptr_t)a.x[w] % 16 == 0 && a.xs[w].b % 8 == 0 && a.xs[w].s % 8 == 0 && a.xs[w].h % 8 == 0;
    const bool four = rows_per_thread(a.c, a.S) == 4;
    if (a.c.D == 128) return four ? append_t<128, 4>(a, vec, st) : append_t<128, 1>(a, vec, st);
    return four ? append_t<64, 4>(a, vec, st) : append_t<64, 1>(a, vec, st);
}

cudaError_t launch_kv4_read(const Kv4ReadArgs& a, cudaStream_t st) {
    const bool four = rows_per_thread(a.c, a.S) == 4;
    if (a.c.D == 128) return four ? read_t<128, 4>(a, st) : read_t<128, 1>(a, st);
    return four ? read_t<64, 4>(a, st) : read_t<64, 1>(a, st);
}

}  // namespace qw
