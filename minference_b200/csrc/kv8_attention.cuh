// Arguments shared by the kernels of the attention over an 8-bit cache (kv8_attention.cu, kv8_attention_wide.cu).
#pragma once
#include "kv8.cuh"

namespace minf {

constexpr int kSMs = 148;

struct Kv8AttnArgs {
    minf_kv8_cache c;
    const __nv_bfloat16* q;
    long long qs[3];
    __nv_bfloat16* o;
    long long os[3];
    int group, n_q, rows;           // rows = group * n_q per cache head; row r is query head r / n_q, token r % n_q
    const int32_t* lengths;
    int length_all, max_length;
    float scale_log2;
    int splits;                     // wide kernel: parts of a head's tokens; narrow kernel: CTAs in all
    int cluster;                    // narrow kernel: CTAs of a head, which join their parts themselves; 0: all CTAs share all heads
    float* part_o;                  // results of parts, normalised, fp32 [..][128]: wide [batch*heads*rows][splits], narrow [piece][rows]
    float* part_lse;                // their log-sum-exps
    float* lse;                     // caller's, [batch, hq, n_q], or NULL
    float* row_lse;                 // [batch*heads*rows] (for the weights), or NULL
    float* logits;                  // [batch*heads][tokens][pitch], or NULL
    int pitch;
    long long tokens;               // rows of `logits` per head
    int chunk;                      // tokens of a CTA that sums weights
    float* weights;
    long long ws[2];
    const float* add_to;
    long long as[2];
};

constexpr int kWideRows = 128;      // query rows of a CTA of the wide kernel
cudaError_t launch_attention_wide(const Kv8AttnArgs& a, int tiles, cudaStream_t stream);

}  // namespace minf
