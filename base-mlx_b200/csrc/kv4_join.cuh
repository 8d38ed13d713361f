// Joining the partials of a row whose keys were split: (base exponent m, sum l,
// output o[D]) each, relative to 2^m.
#pragma once
#include "kv4_tile.cuh"

namespace qw {
namespace kv4 {

// The WPR warps of a row take its n partials in turn; slot(k) is partial k's row in `part` and `pml`,
// or negative if it was left empty.  The caller's warps are `wi` of the row (all of them or none take part);
// `sh` is shared memory of WPR x (D + 2) floats per row; UNROLL partials are in flight at a time.  Lane l holds dimensions l D / 32 ...
template <int D, int WPR, int UNROLL, typename Slot>
QW_DEV void join_row(int n, int wi, Slot slot, const float* part, const float2* pml, float* sh, bf16* dst, float* lse) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31;
    float M = M0, l = 0.f, o[V];
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.f;
    for (int k0 = wi; k0 < n; k0 += 32 * WPR) {
        // this warp's next 32 partials, one per lane
        const int k = k0 + lane * WPR;
        const long long s = k < n ? slot(k) : -1;
        const float2 ml = s >= 0 ? pml[s] : make_float2(M0, 0.f);
        const float m = fmaxf(M, warp_max(ml.x)), al = half_pow(M - m), f = s >= 0 ? half_pow(ml.x - m) : 0.f;
        l = fmaf(l * al, al, warp_sum(ml.y * f * f));
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = o[e] * al * al;
        M = m;
        const int cnt = min(32, (n - k0 + WPR - 1) / WPR);
        for (int j = 0; j < cnt; j += UNROLL) {
            float v[UNROLL][V];
#pragma unroll
            for (int e = 0; e < UNROLL; ++e) {
                const long long t = __shfl_sync(0xffffffffu, s, min(j + e, 31));
                const bool in = j + e < cnt && t >= 0;
                const float* p = part + (in ? (size_t)t * D : 0) + lane * V;
                if (V == 4) {
                    const float4 u = in ? *reinterpret_cast<const float4*>(p) : make_float4(0.f, 0.f, 0.f, 0.f);
                    v[e][0] = u.x, v[e][1] = u.y, v[e][V - 2] = u.z, v[e][V - 1] = u.w;
                } else {
                    const float2 u = in ? *reinterpret_cast<const float2*>(p) : make_float2(0.f, 0.f);
                    v[e][0] = u.x, v[e][1] = u.y;
                }
            }
#pragma unroll
            for (int e = 0; e < UNROLL; ++e) {
                const float fe = j + e < cnt ? __shfl_sync(0xffffffffu, f, min(j + e, 31)) : 0.f;
#pragma unroll
                for (int d = 0; d < V; ++d) o[d] = fmaf(v[e][d] * fe, fe, o[d]);
            }
        }
    }
    if (WPR > 1) {
        float* mine = sh + wi * (D + 2);
        if (lane == 0) {
            mine[D] = M;
            mine[D + 1] = l;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) mine[lane * V + e] = o[e];
        __syncthreads();
        if (wi != 0) return;
#pragma unroll
        for (int w = 1; w < WPR; ++w) M = fmaxf(M, sh[w * (D + 2) + D]);
        l = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) {
            const float* p = sh + w * (D + 2);
            const float f = half_pow(p[D] - M);
            l = fmaf(p[D + 1] * f, f, l);
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = fmaf(p[lane * V + e] * f, f, o[e]);
        }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int e = 0; e < V; e += 2)
        *reinterpret_cast<uint32_t*>(dst + lane * V + e) = l != 0.f ? pack_bf16x2(o[e] * inv, o[e + 1] * inv) : 0u;
    if (lse && lane == 0) *lse = l != 0.f ? (M + log2f(l)) * LN2 : -INFINITY;
}

}  // namespace kv4
}  // namespace qw
