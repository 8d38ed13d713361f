// Writing rows into the 4-bit KV cache and reading them back.
//
// Quantisation of a group x[0..63] of a bf16 row (the format of the model
// weights): bias = min x, scale = bf16((max x - min x) / 15),
// q = clamp(round_half_even((x - bias) / scale), 0, 15), q = 0 where scale = 0.
// A group that holds a NaN or an infinity gets scale = bias = NaN, so all of
// it reads back as NaN.
//
// Every q is the rounding of the exact quotient: the fp32 quotient (error below
// 3e-6 for values up to 16) decides unless it lies within 1e-5 of a half, and
// the few that do are redone in fp64.
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
    float s = __fdiv_rn(d, 15.0f);
    // next to a midpoint of two bf16 values (or past the fp32 range) the fp32 steps may decide wrongly
    const uint32_t low = __float_as_uint(s) & 0xFFFFu;
    if (!(d <= 3.0e38f) || (low >= 0x7FF8u && low <= 0x8008u))
        s = __double2float_rn(((double)hi - (double)lo) / 15.0);
    return bfr(s);
}

QW_DEV uint32_t quantize(float x, float bias, float scale, float inv) {
    float t = __fmul_rn(__fsub_rn(x, bias), inv);
    float r = rintf(t);
    if (!(fabsf(t - r) < 0.49999f))  // also taken for an overflowed quotient
        r = (float)rint(((double)x - (double)bias) / (double)scale);
    return (uint32_t)fminf(fmaxf(r, 0.f), 15.f);
}

// CTA = one (sequence, K or V, head) and NT / TPR consecutive new rows.
template <int D, bool VEC>
__global__ void __launch_bounds__(NT) kv4_append_kernel(const Kv4StoreArgs a) {
    constexpr int T = TPR<D>;
    const int which = blockIdx.y / a.c.heads, h = blockIdx.y % a.c.heads, b = blockIdx.z;
    const int i = blockIdx.x * (NT / T) + threadIdx.x / T, e = threadIdx.x % T;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, a.err,
                                blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0);
    const bool live = i < rw.n;
    float x[8];
    if (live) {
        const bf16* src = a.x[which] + (b * a.xs[which].b + i * a.xs[which].s + h * a.xs[which].h) + e * 8;
        if (VEC) {
            const uint4 u = *reinterpret_cast<const uint4*>(src);
            const uint32_t X[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[2 * j] = bits_lo_f(X[j]);
                x[2 * j + 1] = bits_hi_f(X[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = bf2f(src[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
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
    if (!live) return;
    const bool bad = !(hi <= 3.4e38f) || !(lo >= -3.4e38f);
    float scale = 0.f;
    uint32_t word = 0;
    if (!bad) {
        scale = group_scale(hi, lo);
        if (scale != 0.f) {
            const float inv = __fdiv_rn(1.0f, scale);
#pragma unroll
            for (int j = 0; j < 8; ++j) word |= quantize(x[j], lo, scale, inv) << (4 * j);
        }
    }
    const Kv4Part& p = a.c.p[which];
    const size_t row = ((size_t)b * a.c.heads + h) * a.c.max_pos + (size_t)(rw.off + i);
    p.w[row * T + e] = word;
    if (e % 8 == 0) {
        uint16_t* s = reinterpret_cast<uint16_t*>(p.s) + row * (D / 64) + e / 8;
        uint16_t* z = reinterpret_cast<uint16_t*>(p.b) + row * (D / 64) + e / 8;
        *s = bad ? (uint16_t)0x7FC0 : f_to_bf16bits(scale);
        *z = bad ? (uint16_t)0x7FC0 : f_to_bf16bits(lo);
    }
}

template <int D>
__global__ void __launch_bounds__(NT) kv4_read_kernel(const Kv4ReadArgs a) {
    constexpr int T = TPR<D>;
    const int which = blockIdx.y / a.c.heads, h = blockIdx.y % a.c.heads, b = blockIdx.z;
    const int i = blockIdx.x * (NT / T) + threadIdx.x / T, e = threadIdx.x % T;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, a.err,
                                blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0);
    if (i >= a.S || a.y[which] == nullptr) return;
    uint32_t o[4] = {0u, 0u, 0u, 0u};
    if (i < rw.n) {
        const Kv4Part& p = a.c.p[which];
        const size_t row = ((size_t)b * a.c.heads + h) * a.c.max_pos + (size_t)(rw.off + i);
        const uint32_t w = p.w[row * T + e];
        const float s = bf2f(p.s[row * (D / 64) + e / 8]), z = bf2f(p.b[row * (D / 64) + e / 8]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            o[j] = pack_bf16x2(fmaf(s, (float)((w >> (8 * j)) & 15u), z), fmaf(s, (float)((w >> (8 * j + 4)) & 15u), z));
    }
    bf16* dst = a.y[which] + (((size_t)b * a.S + i) * a.c.heads + h) * D + e * 8;
    *reinterpret_cast<uint4*>(dst) = make_uint4(o[0], o[1], o[2], o[3]);
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4StoreArgs& a, cudaStream_t st) {
    bool vec = true;
    for (int w = 0; w < 2; ++w)
        vec = vec && (uintptr_t)a.x[w] % 16 == 0 && a.xs[w].b % 8 == 0 && a.xs[w].s % 8 == 0 && a.xs[w].h % 8 == 0;
    const int rows = NT / (a.c.D / 8);
    const dim3 grid((a.S + rows - 1) / rows, 2 * a.c.heads, a.c.batch);
    if (a.c.D == 128)
        vec ? kv4_append_kernel<128, true><<<grid, NT, 0, st>>>(a) : kv4_append_kernel<128, false><<<grid, NT, 0, st>>>(a);
    else
        vec ? kv4_append_kernel<64, true><<<grid, NT, 0, st>>>(a) : kv4_append_kernel<64, false><<<grid, NT, 0, st>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_kv4_read(const Kv4ReadArgs& a, cudaStream_t st) {
    const int rows = NT / (a.c.D / 8);
    const dim3 grid((a.S + rows - 1) / rows, 2 * a.c.heads, a.c.batch);
    if (a.c.D == 128)
        kv4_read_kernel<128><<<grid, NT, 0, st>>>(a);
    else
        kv4_read_kernel<64><<<grid, NT, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace qw
