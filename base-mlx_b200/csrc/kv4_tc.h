// The tcgen05 form of the 4-bit cache attention (kv4_attn_tc.cu), chosen by
// kv4_attn.cu for many columns per kv head.
#pragma once
#include "kv4.h"

namespace qw {

struct TcShape {
    int nb, ncb, nsplit;  // 128-column blocks per thread block, blocks of nb * 128 columns, splits of the keys
    size_t part_rows;  // partial rows (D floats and a float2 each) the splits leave
};
TcShape kv4_tc_shape(const Kv4View& c, int S, int Hq, int num_sms);
cudaError_t launch_kv4_attn_tc(const Kv4AttnArgs& a, const TcShape& s, float* part, float2* ml, cudaStream_t st);

}  // namespace qw
