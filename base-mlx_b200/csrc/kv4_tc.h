// The tcgen05 form of the 4-bit cache attention (kv4_attn_tc.cu), chosen by
// kv4_attn.cu for many columns per kv head.
#pragma once
#include "kv4.h"

namespace qw {

struct TcShape {
    int nb, ncb, nsplit;  // 128-column blocks per thread block, blocks of nb * 128 columns, splits of the keys
    size_t part_rows;   // partial rows (D floats and a float2 each) the splits leave
    size_t kept_bytes;  // Q operands [batch][kv head][nb * ncb] of q_block_bytes, then 128 score factors each
};
TcShape kv4_tc_shape(const Kv4View& c, int S, int Hq, int num_sms);
cudaError_t launch_kv4_attn_tc(const Kv4AttnArgs& a, const TcShape& s, float* part, float2* ml, void* kept, cudaStream_t st);
// The weights of such a call, from the Q operands that its attention kernel kept (kv4_mass_tc.cu).
cudaError_t launch_kv4_mass_tc(const Kv4AttnArgs& a, const TcShape& s, const unsigned char* kept, cudaStream_t st);

}  // namespace qw
