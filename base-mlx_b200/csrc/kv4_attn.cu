// Attention over the 4-bit KV cache, optionally accumulating each key's
// attention weight.
//
// Row i of sequence b (n_b new rows behind off_b cached positions, T_b = off_b +
// n_b) and query head h see the keys j < T_b of kv head h / G, with `causal`
// only j <= off_b + i:
//   s_j = scale <q, k_j>, lse = log sum_j exp(s_j), out = sum_j exp(s_j - lse) v_j,
//   mass[b][kv head][j] += sum over the rows and the kv head's query heads of exp(s_j - lse).
// A row that sees no key (a row past n_b, or an empty sequence) gives out = 0, lse = -inf.
#include "kv4.h"

namespace qw {
namespace {

// One warp per (sequence, row, query head); lane l holds the dimensions
// [l * D / 32, (l + 1) * D / 32).  One pass over the keys with a running
// maximum and sum in fp32.
template <int D>
__global__ void __launch_bounds__(128) kv4_attn_row_kernel(const Kv4AttnArgs a) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (long long)a.c.batch * a.S * a.Hq) return;
    const int h = (int)(item % a.Hq), i = (int)(item / a.Hq % a.S), b = (int)(item / a.Hq / a.S);
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, a.err, h == 0 && i == 0 && lane == 0);
    const int vis = i >= rw.n ? 0 : (a.causal ? rw.off + i + 1 : rw.off + rw.n);
    const int kvh = h / (a.Hq / a.c.heads);
    const size_t row0 = ((size_t)b * a.c.heads + kvh) * a.c.max_pos;
    const bf16* qp = a.q + (b * a.qs.b + i * a.qs.s + h * a.qs.h) + lane * V;
    float q[V], o[V], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        q[e] = bf2f(qp[e]) * a.scale;
        o[e] = 0.f;
    }
    const int word = lane * V / 8, sh = 4 * (lane * V % 8), g = lane * V / 64;
    for (int j = 0; j < vis; ++j) {
        const size_t r = row0 + j;
        const uint32_t kw = a.c.p[0].w[r * (D / 8) + word] >> sh, vw = a.c.p[1].w[r * (D / 8) + word] >> sh;
        const float ks = bf2f(a.c.p[0].s[r * (D / 64) + g]), kb = bf2f(a.c.p[0].b[r * (D / 64) + g]);
        const float vs = bf2f(a.c.p[1].s[r * (D / 64) + g]), vb = bf2f(a.c.p[1].b[r * (D / 64) + g]);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) s = fmaf(q[e], fmaf(ks, (float)((kw >> (4 * e)) & 15u), kb), s);
        s = warp_sum(s);
        const float mn = fmaxf(m, s);
        const float al = m == mn ? 1.f : expf(m - mn), p = s == mn ? 1.f : expf(s - mn);
        l = fmaf(l, al, p);
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = fmaf(o[e], al, p * fmaf(vs, (float)((vw >> (4 * e)) & 15u), vb));
        m = mn;
    }
    bf16* op = a.out + (b * a.os.b + i * a.os.s + h * a.os.h) + lane * V;
#pragma unroll
    for (int e = 0; e < V; ++e) op[e] = f2bf(vis > 0 ? o[e] / l : 0.f);
    if (a.lse && lane == 0) a.lse[((size_t)b * a.S + i) * a.Hq + h] = vis > 0 ? m + logf(l) : -INFINITY;
}

// One warp per (sequence, kv head, key): the key's probability summed over the
// rows and query heads in a fixed order.
template <int D>
__global__ void __launch_bounds__(128) kv4_mass_row_kernel(const Kv4AttnArgs a) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    const int j = blockIdx.x * 4 + (threadIdx.x >> 5), kvh = blockIdx.y, b = blockIdx.z;
    const Kv4Rows rw = kv4_rows(a.seq_len, a.n_new, b, a.S, a.c.max_pos, nullptr, false);
    if (j >= rw.off + rw.n) return;
    const size_t r = ((size_t)b * a.c.heads + kvh) * a.c.max_pos + j;
    const int word = lane * V / 8, sh = 4 * (lane * V % 8), g = lane * V / 64, G = a.Hq / a.c.heads;
    const uint32_t kw = a.c.p[0].w[r * (D / 8) + word] >> sh;
    const float ks = bf2f(a.c.p[0].s[r * (D / 64) + g]), kb = bf2f(a.c.p[0].b[r * (D / 64) + g]);
    float k[V], acc = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) k[e] = fmaf(ks, (float)((kw >> (4 * e)) & 15u), kb);
    for (int i = a.causal ? max(0, j - rw.off) : 0; i < rw.n; ++i)
        for (int h = kvh * G; h < (kvh + 1) * G; ++h) {
            const bf16* qp = a.q + (b * a.qs.b + i * a.qs.s + h * a.qs.h) + lane * V;
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) s = fmaf(bf2f(qp[e]) * a.scale, k[e], s);
            s = warp_sum(s);
            acc += expf(s - a.lse[((size_t)b * a.S + i) * a.Hq + h]);
        }
    if (lane == 0) a.mass[r] += acc;
}

}  // namespace

size_t kv4_attn_scratch_bytes(const Kv4View& c, int S, int Hq, int) { return (size_t)c.batch * S * Hq * sizeof(float); }

cudaError_t launch_kv4_attention(const Kv4AttnArgs& in, void* scratch, int, cudaStream_t st) {
    Kv4AttnArgs a = in;
    if (a.mass && !a.lse) a.lse = static_cast<float*>(scratch);
    const long long items = (long long)a.c.batch * a.S * a.Hq;
    const unsigned blocks = (unsigned)((items + 3) / 4);
    if (a.c.D == 128)
        kv4_attn_row_kernel<128><<<blocks, 128, 0, st>>>(a);
    else
        kv4_attn_row_kernel<64><<<blocks, 128, 0, st>>>(a);
    if (a.mass) {
        const dim3 grid((a.c.max_pos + 3) / 4, a.c.heads, a.c.batch);
        if (a.c.D == 128)
            kv4_mass_row_kernel<128><<<grid, 128, 0, st>>>(a);
        else
            kv4_mass_row_kernel<64><<<grid, 128, 0, st>>>(a);
    }
    return cudaGetLastError();
}

}  // namespace qw
