// 4-bit KV cache operators: launch interface shared by capi.cu and the kv4*.cu
// kernel files.
//
// The cache holds every K and V row [sequence][kv head][position] in the MLX
// affine format of the model weights: head_dim / 8 uint32 words (element e at
// bits 4 * (e % 8) of word e / 8) and one bf16 scale and bias per 64 elements,
// value = scale * q + bias.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace qw {

// Words, scales and biases of K (index 0) or V (index 1).
struct Kv4Part {
    uint32_t* w;  // [batch][heads][max_pos][D / 8]
    bf16* s;      // [batch][heads][max_pos][D / 64]
    bf16* b;
};

struct Kv4View {
    Kv4Part p[2];
    int batch, heads, max_pos, D;
};

// Element strides of a [batch][row][head][D] tensor whose last dimension is contiguous.
struct Kv4Strides {
    long long b, s, h;
};

struct Kv4StoreArgs {
    Kv4View c;
    const bf16* x[2];  // K rows, V rows
    Kv4Strides xs[2];
    int S;
    const int* seq_len;  // [batch] first position of the new rows
    const int* n_new;    // [batch] rows to store (at most S), or null: S
    int* err;            // optional error bits
};
cudaError_t launch_kv4_append(const Kv4StoreArgs& a, cudaStream_t st);

struct Kv4ReadArgs {
    Kv4View c;
    bf16* y[2];  // contiguous [batch][S][heads][D]; either may be null
    int S;
    const int* seq_len;  // [batch] first position read, or null: 0
    const int* n_new;    // [batch] rows read, the others are written as zero; or null: S
    int* err;
};
cudaError_t launch_kv4_read(const Kv4ReadArgs& a, cudaStream_t st);

struct Kv4AttnArgs {
    Kv4View c;
    const bf16* q;  // [batch][S][heads][D]
    Kv4Strides qs;
    bf16* out;
    Kv4Strides os;
    int S, Hq, causal;
    float scale;
    const int* seq_len;  // [batch] positions cached before the S new rows
    const int* n_new;    // [batch] new rows (at most S), or null: S
    float* lse;          // [batch][S][Hq]: the caller's, or (mass only) scratch; or null
    float* mass;         // [batch][kv heads][max_pos], added to; or null
    int* err;
};
size_t kv4_attn_scratch_bytes(const Kv4View& c, int S, int Hq, int num_sms);
cudaError_t launch_kv4_attention(const Kv4AttnArgs& a, void* scratch, int num_sms, cudaStream_t st);

struct Kv4EvictArgs {
    Kv4View src, dst;  // the same buffers: in place
    const float* mass_src;  // [batch][heads][src.max_pos]
    float* mass_dst;        // [batch][heads][dst.max_pos]
    const int* seq_len;
    int* new_len;           // [batch]; may be seq_len
    int keep, recent;
    int* index_out;         // [batch][heads][keep], or null
};
size_t kv4_evict_scratch_bytes(const Kv4View& src, int keep);
cudaError_t launch_kv4_evict(const Kv4EvictArgs& a, void* scratch, cudaStream_t st);

// Sequence b's rows of a step of S rows: positions [off, off + n).  Rows past
// max_pos are left out and reported as QW_DERR_KV_RANGE; a length outside
// [0, max_pos] is reported and counts as an empty sequence without rows.
struct Kv4Rows {
    int off, n;
};
QW_DEV Kv4Rows kv4_rows(const int* seq_len, const int* n_new, int b, int S, int max_pos, int* err, bool report) {
    const int off = seq_len ? seq_len[b] : 0;
    const int want = n_new ? max(0, min(n_new[b], S)) : S;
    const bool bad = off < 0 || off > max_pos;
    Kv4Rows r;
    r.off = bad ? 0 : off;
    r.n = bad ? 0 : min(want, max_pos - off);
    if (report && err && (bad || want > r.n)) atomicOr(err, (int)QW_DERR_KV_RANGE);
    return r;
}

}  // namespace qw
