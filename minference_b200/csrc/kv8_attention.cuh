// Arguments shared by the kernels of the attention over an 8-bit cache (kv8_attention.cu, kv8_attention_wide.cu).
#pragma once
#include "kv8.cuh"

namespace minf {

constexpr int kSMs = 148;

// Numerators are kept as f16 kHeadroom powers of two above their value.  The reference they are relative to follows jumps of
// more than 2^8 only, so they reach 2^15 (f16 ends at 65504); a token is rounded to 2^-11 of its numerator down to 2^-21 of the
// largest, and to 2^-32 of the largest below that.  (Without the headroom those were 2^-14 and 2^-25: behind a strong token of no
// value, weak ones 24 bits below it came out wrong by a percent, ones of 26 bits by half.)  Denominators take it out again term
// by term, outputs at the end.
constexpr float kHeadroom = 7.f, kHeadroomOut = 0.0078125f;

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
