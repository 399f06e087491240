// Filling, reading back and shrinking an 8-bit key/value cache (layout: kv8.cuh).
//
// Quantisation of a block x (64 tokens x 128 of one head): with m the largest finite magnitude,
//   e4m3: scale = 2^p, p the smallest with 448 * 2^p >= m -- dividing by a power of two is exact, so a code is the one
//         rounding of x to e4m3's grid, and requantising values that came from codes loses nothing but what falls
//         below the new grid's subnormals;
//   int8: scale = m / 127 in fp32, code = round-half-even(x / scale) with an IEEE division.
// Scales are at least 2^-100; an all-zero block has scale 1.  NaN stays NaN in e4m3 and becomes 0 in int8; infinities
// become the largest code.
#include "kv8.cuh"

#include <cooperative_groups.h>

#include <algorithm>

#include "sm100_ptx.cuh"

namespace minf {

int kv8_check(const minf_kv8_cache* c) {
    if (!c) return fail(MINF_E_ARG, "null cache");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail || !c->status)
        return fail(MINF_E_ARG, "null pointer in the cache");
    if (c->batch < 1 || c->heads < 1 || c->batch > 65535 || c->heads > 32767)
        return fail(MINF_E_ARG, "bad cache sizes (batch %d, heads %d)", c->batch, c->heads);
    if (c->capacity < kKv8Block || c->capacity % kKv8Block || c->capacity > (1 << 30))
        return fail(MINF_E_ARG, "the cache's capacity must be a positive multiple of %d tokens, 2^30 at most (got %d)", kKv8Block, c->capacity);
    if (c->format != MINF_KV8_E4M3 && c->format != MINF_KV8_INT8) return fail(MINF_E_ARG, "unknown cache format %d", c->format);
    const uintptr_t all = reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) |
                          reinterpret_cast<uintptr_t>(c->k_tail) | reinterpret_cast<uintptr_t>(c->v_tail);
    if (all & 15) return fail(MINF_E_ARG, "the cache's tensors must be 16-byte aligned");
    return MINF_OK;
}

// Largest finite magnitude of the block from each thread's own, for all threads of the CTA.
template <int THREADS>
__device__ __forceinline__ float block_max(float m, float* red) {
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) m = fmaxf(m, red[i]);
    return m;
}

__device__ __forceinline__ float finite_magnitude(float x) {
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;          // NaN compares false
}

template <int FMT>
__device__ __forceinline__ float scale_of(float top) {
    if (!(top > 0.f)) return 1.f;
    if constexpr (FMT == MINF_KV8_E4M3) {
        int e;
        const float m = frexpf(top, &e);    // top = m * 2^e, 0.5 <= m < 1;  448 = 0.875 * 2^9
        return __uint_as_float((uint32_t)(max(m <= 0.875f ? e - 9 : e - 8, -100) + 127) << 23);     // (p is 120 at most)
    } else {
        return fmaxf(__fdiv_rn(top, 127.f), kKv8MinScale);
    }
}

template <int FMT>
__device__ __forceinline__ uint2 values_to_codes(const float (&x)[8], float scale) {
    uint32_t c[2];
    if constexpr (FMT == MINF_KV8_E4M3) {
        const float inv = __fdiv_rn(1.f, scale);            // a power of two: exact
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint16_t lo, hi;
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[4 * i + 1] * inv), "f"(x[4 * i] * inv));
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[4 * i + 3] * inv), "f"(x[4 * i + 2] * inv));
            c[i] = (uint32_t)lo | ((uint32_t)hi << 16);
        }
    } else {
        // x / scale rounded to an integer: by the reciprocal, which is right unless the quotient lies next to a half (both
        // quotients' errors together are below 127 * 2^-23), and there by the division the definition has.  Adding 1.5 * 2^23
        // rounds to the nearest integer and leaves it in the low bits.
        constexpr float kRound = 12582912.f;
        const float inv = __fdiv_rn(1.f, scale);
        bool sure = true;                                   // (false for what is not finite too)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float t = __fmaf_rn(x[4 * i + j], inv, kRound);
                sure = sure && fabsf(__fmaf_rn(x[4 * i + j], inv, -(t - kRound))) < 0.49998f;
                q[j] = __float_as_uint(t);
            }
            c[i] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
        }
        if (!sure) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t w = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float q = rintf(__fdiv_rn(x[4 * i + j], scale));
                    const int r = q != q ? 0 : (int)fminf(fmaxf(q, -127.f), 127.f);
                    w |= (uint32_t)(r & 0xff) << (8 * j);
                }
                c[i] = w;
            }
        }
    }
    return make_uint2(c[0], c[1]);
}

// ------------------------------------------------------------------------------------------------- store
// One CTA per (block of 64 tokens that gets new ones, head, keys or values).  256 threads hold the block in
// registers, sixteen values of two rows each: one read of the new tokens, one write of the codes.
// Bound by HBM for e4m3: 4 B read and 2 B written per (key, value) pair of elements; 131072 tokens of 8 heads (537 MB read,
// 268 MB written) take 123 us, 6.5 TB/s.  int8 takes 187 us, 4.3 TB/s: its rounding and its search for quotients next to a half
// keep the issue slots 75 % busy.
struct StoreArgs {
    minf_kv8_cache c;
    const __nv_bfloat16* src[2];
    long long stride[2][3];
    int n_tokens;
    const int32_t* start;
    int start_all;
    const int32_t* counts;
};

constexpr int kStoreThreads = 256;

template <int FMT>
__global__ void __launch_bounds__(kStoreThreads) kv8_store_kernel(const __grid_constant__ StoreArgs a) {
    __shared__ float red[kStoreThreads / 32];
    const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1;
    const int start = a.start ? a.start[b] : a.start_all;
    const int count = a.counts ? a.counts[b] : a.n_tokens;
    if (start < 0 || count < 0 || count > a.n_tokens || start > a.c.capacity - count) {
        if (threadIdx.x == 0) atomicOr(a.c.status + MINF_ST_ERROR, MINF_ERR_KV8_RANGE);
        return;                                             // nothing of this sequence is stored
    }
    if (count == 0) return;
    const int end = start + count;
    const int blk0 = start / kKv8Block, last = (end - 1) / kKv8Block;
    const int blk = blk0 + blockIdx.x;
    if (blk > last) return;
    const bool complete = (blk + 1) * kKv8Block <= end;
    if (!complete && blk != blk0) return;                   // the first block's CTA writes the tail once it has read it
    const size_t bh = (size_t)b * a.c.heads + h;
    const __nv_bfloat16* src = a.src[which] + b * a.stride[which][0] + h * a.stride[which][1];
    const long long row_stride = a.stride[which][2];
    __nv_bfloat16* tail = static_cast<__nv_bfloat16*>(which ? a.c.v_tail : a.c.k_tail) + bh * (kKv8Block * kKv8Dim);
    const int chunk = threadIdx.x & 7, row0 = threadIdx.x >> 3;        // 16 values of rows row0 and row0 + 32
    auto new_row = [&](int t) { return reinterpret_cast<const uint4*>(src + (t - start) * row_stride + chunk * 16); };
    auto tail_row = [&](int r) { return reinterpret_cast<uint4*>(tail + r * kKv8Dim + chunk * 16); };

    if (complete) {
        uint4 raw[2][2];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = row0 + 32 * i, t = blk * kKv8Block + r;
            if (t < start) {
                raw[i][0] = tail_row(r)[0];
                raw[i][1] = tail_row(r)[1];
            } else {
                raw[i][0] = __ldcs(new_row(t));
                raw[i][1] = __ldcs(new_row(t) + 1);
            }
        }
        // the largest magnitude two values at a time (NaN is passed over); only if it is infinite, the finite ones one by one
        __nv_bfloat162 top2 = __float2bfloat162_rn(0.f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4& x = raw[i >> 1][i & 1];
            const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t m = words[j] & 0x7fff7fffu;
                top2 = __hmax2(top2, *reinterpret_cast<const __nv_bfloat162*>(&m));
            }
        }
        top = block_max<kStoreThreads>(fmaxf(__low2float(top2), __high2float(top2)), red);     // (its barrier also ends the reads of the tail)
        if (top == INFINITY) {                              // the same in every thread
            top = 0.f;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                float x[8];
                bf16x8_to_values(raw[i >> 1][i & 1], x);
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, finite_magnitude(x[j]));
            }
            __syncthreads();
            top = block_max<kStoreThreads>(top, red);
        }
        const float scale = scale_of<FMT>(top);
        uint8_t* codes = static_cast<uint8_t*>(which ? a.c.v : a.c.k) + (bh * a.c.capacity + (size_t)blk * kKv8Block) * kKv8Dim;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float x[8], y[8];
            bf16x8_to_values(raw[i][0], x);
            bf16x8_to_values(raw[i][1], y);
            const uint2 lo = values_to_codes<FMT>(x, scale), hi = values_to_codes<FMT>(y, scale);
            *reinterpret_cast<uint4*>(codes + (row0 + 32 * i) * kKv8Dim + chunk * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        if (threadIdx.x == 0) (which ? a.c.v_scale : a.c.k_scale)[bh * (a.c.capacity / kKv8Block) + blk] = scale;
    }
    if (blk == blk0 && end % kKv8Block) {                   // the tokens behind the last complete block
        const int t0 = max(start, last * kKv8Block);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = last * kKv8Block + row0 + 32 * i;
            if (t >= t0 && t < end) {
                tail_row(row0 + 32 * i)[0] = new_row(t)[0];
                tail_row(row0 + 32 * i)[1] = new_row(t)[1];
            }
        }
    }
}

// -------------------------------------------------------------------------------------------------- load
// One CTA per (64 tokens, head, keys or values), sixteen values of two rows a thread.  Bound by HBM, one byte read for two
// written: 131072 tokens of 8 heads take 126-128 us of either type, 6.4 TB/s.
struct LoadArgs {
    minf_kv8_cache c;
    const int32_t* lengths;
    int length_all;
    const int32_t* first;
    int first_all;
    int count;
    __nv_bfloat16* out[2];
};

__device__ __forceinline__ uint4 pack_bf16x8(const float (&v)[8]) {
    return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}

template <int FMT>
__global__ void __launch_bounds__(kStoreThreads) kv8_load_kernel(const __grid_constant__ LoadArgs a) {
    const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1;
    const int n = kv8_length(a.lengths, a.length_all, b, a.c.capacity, a.c.status);
    const long long first = a.first ? a.first[b] : a.first_all;
    const size_t bh = (size_t)b * a.c.heads + h;
    const int chunk = threadIdx.x & 7;                      // 16 values of two rows
    const int whole = n / kKv8Block * kKv8Block;
    const uint8_t* codes = static_cast<const uint8_t*>(which ? a.c.v : a.c.k) + bh * a.c.capacity * kKv8Dim + chunk * 16;
    const float* scales = (which ? a.c.v_scale : a.c.k_scale) + bh * (a.c.capacity / kKv8Block);
    const __nv_bfloat16* tail = static_cast<const __nv_bfloat16*>(which ? a.c.v_tail : a.c.k_tail) + bh * (kKv8Block * kKv8Dim) + chunk * 16;
    __nv_bfloat16* out = a.out[which] + bh * a.count * kKv8Dim + chunk * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = blockIdx.x * kKv8Block + (threadIdx.x >> 3) + 32 * i;
        if (r >= a.count) break;
        const long long t = first + r;
        uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
        if (t >= 0 && t < whole) {
            const uint4 c = *reinterpret_cast<const uint4*>(codes + (size_t)t * kKv8Dim);
            const float scale = scales[t / kKv8Block];
            float v[8];
            codes_to_values<FMT>(make_uint2(c.x, c.y), scale, v);
            lo = pack_bf16x8(v);
            codes_to_values<FMT>(make_uint2(c.z, c.w), scale, v);
            hi = pack_bf16x8(v);
        } else if (t >= whole && t < n) {
            const uint4* x = reinterpret_cast<const uint4*>(tail + (t - whole) * kKv8Dim);
            lo = x[0];
            hi = x[1];
        }
        uint4* to = reinterpret_cast<uint4*>(out + (size_t)r * kKv8Dim);
        to[0] = lo;
        to[1] = hi;
    }
}

// ------------------------------------------------------------------------------------------------- evict
struct SelectArgsKv8 {
    minf_kv8_cache c;               // the source
    const int32_t* lengths;
    int length_all, max_length;
    const float* weights;           // [batch, heads, >= max_length] with the strides below, tokens contiguous
    long long w_stride[2];
    int budget, recent, sink;
    int cached;                     // keys a CTA has room for
    int32_t* kept;                  // [batch, heads, budget]
};

// Weights in the order of their keys: larger weight, larger key; -0 equals 0, a NaN is the largest.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.f);            // -0 + 0 = 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kSelectCluster = 8;                           // CTAs at most that share a head's tokens
constexpr int kSelectPart = 8192;                           // tokens from which on one more is worth its barriers
constexpr int kSelectBins = 2048;
constexpr int kSelectList = 2048;                           // keys of the first two passes' bin that a CTA lists
constexpr int kSelectCached = 40960;                        // keys a CTA keeps in shared memory at most
// shared memory in words: two histograms (of the even and the odd lanes), the cluster's sums of three passes, the list, the keys
constexpr int kSelectWords = 2 * kSelectBins + 3 * kSelectBins + kSelectList;

// A cluster per (sequence, head), each CTA a contiguous part of the candidates, whose keys it reads once and keeps in
// shared memory (beyond 8 x 40960 candidates it reads them again from L2 in each pass).  Three passes of 11, 11 and 10
// bits find the key of the last token that is kept: every CTA adds the bins it has to the first one's sums, which finds
// the digit for all.  (Every CTA summing all histograms by itself moved 64 KB through distributed shared memory a pass:
// 4800 cycles instead of 1300 and a barrier.)  Then the warps, each with a contiguous stretch, count what they keep and
// write it at the offset of everything before them: ascending order without a sort, equal keys by position.
// What bounds it at 131072 tokens: the first pass (4 B a token read, atomics on a few dozen hot bins) and seven barriers
// across the cluster of 1500 cycles each: 24 us for 8 heads (30 with cold caches), 16 us (19) for 32 heads of 9000 tokens.  Four
// histograms a CTA instead of two gain 1 us there and lose 1 us here.  ptxas gives it 32 registers and 20 bytes of spills.
__global__ void __launch_bounds__(kSelectThreads) kv8_select_kernel(const __grid_constant__ SelectArgsKv8 a) {
    extern __shared__ uint32_t dyn[];
    uint32_t* hist = dyn;
    uint32_t* sums = dyn + 2 * kSelectBins;
    uint32_t* list = sums + 3 * kSelectBins;
    uint32_t* cached = dyn + kSelectWords;
    __shared__ uint32_t warp_sum[kSelectWarps];
    __shared__ uint32_t sh_digit[3], sh_need[3], listed;
    __shared__ uint32_t warp_above[kSelectWarps], warp_equal[kSelectWarps];
    __shared__ uint32_t cta_above, cta_equal;
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = cluster.num_blocks(), part = blockIdx.x % parts, h = blockIdx.x / parts, b = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = kv8_length(a.lengths, a.length_all, b, a.max_length, a.c.status);
    dependents_launch();
    const float* w = a.weights + b * a.w_stride[0] + h * a.w_stride[1];
    int32_t* kept = a.kept + ((size_t)b * a.c.heads + h) * a.budget;
    if (n <= a.budget) {                                    // everything stays (the whole cluster leaves here)
        for (int i = part * kSelectThreads + tid; i < a.budget; i += parts * kSelectThreads) kept[i] = i < n ? i : -1;
        return;
    }
    const int lo = a.sink, hi = n - a.recent;
    for (int i = part * kSelectThreads + tid; i < a.sink + a.recent; i += parts * kSelectThreads)
        kept[i < a.sink ? i : a.budget - a.recent + (i - a.sink)] = i < a.sink ? i : hi + (i - a.sink);
    uint32_t need = a.budget - a.sink - a.recent;           // of hi - lo > need candidates
    if (need == 0) return;
    const int chunk = ((hi - lo + parts - 1) / parts + 31) / 32 * 32;
    const int c0 = min(hi, lo + part * chunk), c1 = min(hi, c0 + chunk), count = c1 - c0;
    const bool in_smem = count <= a.cached;
    auto key_at = [&](int i) { return in_smem ? cached[i] : weight_key(w[c0 + i]); };
    auto sync = [&] {
        if (parts > 1) cluster.sync();
        else __syncthreads();
    };
    for (int i = tid; i < 3 * kSelectBins; i += kSelectThreads) sums[i] = 0;
    if (tid == 0) listed = 0;
    if (parts > 1) cluster.barrier_arrive();                // the first one's sums are clear before anybody adds to them

    uint32_t prefix = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
        const uint32_t mask = (1u << bits) - 1u;
        for (int i = tid; i < 2 * kSelectBins; i += kSelectThreads) hist[i] = 0;
        __syncthreads();
        auto add = [&](uint32_t key) { atomicAdd(&hist[2 * ((key >> shift) & mask) + (lane & 1)], 1u); };
        if (pass == 2 && listed <= kSelectList) {
            for (int i = tid; i < (int)listed; i += kSelectThreads)
                if (list[i] >> 10 == prefix) add(list[i]);
        } else {
            for (int i0 = 0; i0 < count; i0 += 8 * kSelectThreads) {
                uint32_t key[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int i = i0 + u * kSelectThreads + tid;
                    key[u] = i >= count ? 0u : pass == 0 ? weight_key(w[c0 + i]) : key_at(i);
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int i = i0 + u * kSelectThreads + tid;
                    if (pass == 0) {
                        if (i < count) {
                            if (in_smem) cached[i] = key[u];
                            add(key[u]);
                        }
                    } else {
                        const bool live = i < count && key[u] >> (shift + bits) == prefix;
                        const uint32_t who = __ballot_sync(0xffffffffu, live);
                        if (who == 0) continue;
                        if (live) add(key[u]);
                        if (pass == 1) {                    // for the third pass
                            uint32_t at = 0;
                            if (lane == 0) at = atomicAdd(&listed, __popc(who));
                            at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
                            if (live && at < kSelectList) list[at] = key[u];
                        }
                    }
                }
            }
        }
        __syncthreads();
        if (pass == 0 && parts > 1) cluster.barrier_wait();
        uint32_t* total = sums + pass * kSelectBins;
        uint32_t* to = parts > 1 ? cluster.map_shared_rank(total, 0) : total;
        for (int i = tid; i < kSelectBins; i += kSelectThreads) {
            const uint32_t x = hist[2 * i] + hist[2 * i + 1];
            if (x) atomicAdd(to + i, x);
        }
        sync();
        if (part == 0) {
            // thread t has bins 2046 - 2t and 2047 - 2t: a scan over the threads runs from the largest key down
            const int bin = kSelectBins - 2 - 2 * tid;
            const uint32_t x0 = total[bin], x1 = total[bin + 1];
            uint32_t scan = x0 + x1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, scan, o);
                if (lane >= o) scan += y;
            }
            if (lane == 31) warp_sum[warp] = scan;
            __syncthreads();
            const uint32_t before = scan - x0 - x1 + __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0u);
            if (before < need && need <= before + x1) {
                sh_digit[pass] = bin + 1;
                sh_need[pass] = need - before;
            } else if (before + x1 < need && need <= before + x1 + x0) {
                sh_digit[pass] = bin;
                sh_need[pass] = need - before - x1;
            }
        }
        sync();
        prefix = (prefix << bits) | (parts > 1 ? *cluster.map_shared_rank(&sh_digit[pass], 0) : sh_digit[pass]);
        need = parts > 1 ? *cluster.map_shared_rank(&sh_need[pass], 0) : sh_need[pass];
    }
    // Keys above `prefix` are kept, and the first `need` that equal it.  A warp takes its stretch 32 words of 32 tokens at a
    // time: lane i has the words (above, equal) of tokens 32 i on.
    const int seg = ((count + kSelectWarps - 1) / kSelectWarps + 31) / 32 * 32;
    const int s0 = min(count, warp * seg), s1 = min(count, s0 + seg);
    auto words = [&](int base, uint32_t& gt, uint32_t& eq) {
        gt = eq = 0;
        for (int j = 0; j < 32 && base + 32 * j < s1; ++j) {
            const int i = base + 32 * j + lane;
            const uint32_t k = i < s1 ? key_at(i) : 0u;
            const uint32_t bg = __ballot_sync(0xffffffffu, i < s1 && k > prefix), be = __ballot_sync(0xffffffffu, i < s1 && k == prefix);
            if (lane == j) {
                gt = bg;
                eq = be;
            }
        }
    };
    uint32_t above = 0, equal = 0, first_gt = 0, first_eq = 0;
    for (int base = s0; base < s1; base += 1024) {
        uint32_t gt, eq;
        words(base, gt, eq);
        above += __popc(gt);
        equal += __popc(eq);
        if (base == s0) {
            first_gt = gt;
            first_eq = eq;
        }
    }
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) {
        warp_above[warp] = above;
        warp_equal[warp] = equal;
    }
    __syncthreads();
    if (warp == 0) {
        const uint32_t ca = __reduce_add_sync(0xffffffffu, warp_above[lane]), ce = __reduce_add_sync(0xffffffffu, warp_equal[lane]);
        if (lane == 0) {
            cta_above = ca;
            cta_equal = ce;
        }
    }
    sync();
    // before this warp's stretch: the parts before this one, the warps before this one
    uint32_t gt_before = lane < warp ? warp_above[lane] : 0u, eq_before = lane < warp ? warp_equal[lane] : 0u;
    if (lane < part) {
        gt_before += *cluster.map_shared_rank(&cta_above, lane);
        eq_before += *cluster.map_shared_rank(&cta_equal, lane);
    }
    gt_before = __reduce_add_sync(0xffffffffu, gt_before);
    eq_before = __reduce_add_sync(0xffffffffu, eq_before);
    for (int base = s0; base < s1; base += 1024) {
        uint32_t gt = first_gt, eq = first_eq;
        if (base != s0) words(base, gt, eq);
        uint32_t gs = __popc(gt), es = __popc(eq);          // scans over the lanes' words
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, gs, o), y = __shfl_up_sync(0xffffffffu, es, o);
            if (lane >= o) {
                gs += x;
                es += y;
            }
        }
        uint32_t g = gt_before + gs - __popc(gt), e = eq_before + es - __popc(eq);
        gt_before += __shfl_sync(0xffffffffu, gs, 31);
        eq_before += __shfl_sync(0xffffffffu, es, 31);
        for (uint32_t both = gt | eq; both; both &= both - 1) {
            const int bit = __ffs(both) - 1;
            const bool is_gt = gt >> bit & 1u;
            if (is_gt || e < need) {
                const uint32_t at = a.sink + g + min(e, need);
                if (at < (uint32_t)a.budget) kept[at] = c0 + base + 32 * lane + bit;
            }
            if (is_gt) ++g;
            else ++e;
        }
    }
    sync();                                                 // the counts are read by the others
}

struct GatherArgs {
    minf_kv8_cache src, dst;
    const int32_t* lengths;
    int length_all, max_length;
    const float* weights;
    long long w_stride[2];
    int budget;
    const int32_t* kept;
    float* weights_out;             // [batch, heads, dst.capacity]
    int32_t* lengths_out;
};

// One CTA per (block of the new cache, head, keys or values): the kept tokens' values, quantised again as a block.  Bound by
// two reads one after the other (which token, then its codes): 8-9 us for 8 heads of 4096 tokens, 11 MB (12 with cold caches).
// The six CTAs an SM leave 40 registers a thread, of which int8 spills 8 bytes.
template <int FMT>
__global__ void __launch_bounds__(kStoreThreads, 6) kv8_gather_kernel(const __grid_constant__ GatherArgs a) {
    __shared__ float red[kStoreThreads / 32];
    const int b = blockIdx.z, h = blockIdx.y >> 1, which = blockIdx.y & 1, blk = blockIdx.x;
    const int n = kv8_length(a.lengths, a.length_all, b, a.max_length, a.src.status);
    const int m = min(n, a.budget);
    const size_t bh = (size_t)b * a.src.heads + h;
    const int32_t* kept = a.kept + bh * a.budget;
    dependents_wait();
    if (which == 0 && threadIdx.x < kKv8Block) {
        const int slot = blk * kKv8Block + threadIdx.x;
        float w = 0.f;
        if (slot < m) {
            const int t = kept[slot];
            if (t >= 0 && t < n) w = a.weights[b * a.w_stride[0] + h * a.w_stride[1] + t];
        }
        a.weights_out[bh * a.dst.capacity + slot] = w;
    }
    if (blk == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.lengths_out[b] = m;
    if (blk * kKv8Block >= m) return;
    const bool complete = (blk + 1) * kKv8Block <= m;
    const int chunk = threadIdx.x & 15, row0 = threadIdx.x >> 4;
    // A row's eight values as they lie in the source (codes, or bf16 of the tail) and their scale: turned into numbers
    // twice, for the maximum and for the new codes, because few registers -- many blocks on an SM -- hide the two
    // dependent reads this kernel waits for.
    const int whole = n / kKv8Block * kKv8Block;
    const uint8_t* src_codes = static_cast<const uint8_t*>(which ? a.src.v : a.src.k) + bh * a.src.capacity * kKv8Dim + chunk * 8;
    const __nv_bfloat16* src_tail = static_cast<const __nv_bfloat16*>(which ? a.src.v_tail : a.src.k_tail) + bh * (kKv8Block * kKv8Dim) + chunk * 8;
    const float* src_scale = (which ? a.src.v_scale : a.src.k_scale) + bh * (a.src.capacity / kKv8Block);
    uint4 raw[4];
    float scale_in[4];
    unsigned coded = 0;                                     // bit i: row i is codes, else bf16 (or nothing: zeros)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int slot = blk * kKv8Block + row0 + 16 * i;
        const int t = slot < m ? kept[slot] : -1;
        raw[i] = make_uint4(0u, 0u, 0u, 0u);
        scale_in[i] = 0.f;
        if (t >= 0 && t < whole) {
            const uint2 c = *reinterpret_cast<const uint2*>(src_codes + (size_t)t * kKv8Dim);
            raw[i].x = c.x;
            raw[i].y = c.y;
            scale_in[i] = src_scale[t / kKv8Block];
            coded |= 1u << i;
        } else if (t >= whole && t < n) {
            raw[i] = *reinterpret_cast<const uint4*>(src_tail + (t - whole) * kKv8Dim);
        }
    }
    auto values = [&](int i, float (&x)[8]) {
        if (coded >> i & 1u) codes_to_values<FMT>(make_uint2(raw[i].x, raw[i].y), scale_in[i], x);
        else bf16x8_to_values(raw[i], x);
    };
    if (complete) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float big = INFINITY;
            if (coded >> i & 1u) {                          // the largest code (NaN is passed over) times its scale
                uint32_t h[4];
                codes_to_half<FMT>(raw[i].x, h[0], h[1]);
                codes_to_half<FMT>(raw[i].y, h[2], h[3]);
                __half2 m = __float2half2_rn(0.f);
#pragma unroll
                for (int j = 0; j < 4; ++j) m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&h[j])));
                big = fmaxf(__low2float(m), __high2float(m)) * scale_in[i];
            }
            if (!(big < INFINITY)) {                        // the tail's values, and codes next to fp32's largest
                float x[8];
                values(i, x);
                big = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) big = fmaxf(big, finite_magnitude(x[j]));
            }
            top = fmaxf(top, big);
        }
        top = block_max<kStoreThreads>(top, red);
        const float scale = scale_of<FMT>(top);
        uint8_t* codes = static_cast<uint8_t*>(which ? a.dst.v : a.dst.k) + (bh * a.dst.capacity + (size_t)blk * kKv8Block) * kKv8Dim;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float x[8];
            values(i, x);
            *reinterpret_cast<uint2*>(codes + (row0 + 16 * i) * kKv8Dim + chunk * 8) = values_to_codes<FMT>(x, scale);
        }
        if (threadIdx.x == 0) (which ? a.dst.v_scale : a.dst.k_scale)[bh * (a.dst.capacity / kKv8Block) + blk] = scale;
    } else {
        __nv_bfloat16* tail = static_cast<__nv_bfloat16*>(which ? a.dst.v_tail : a.dst.k_tail) + bh * (kKv8Block * kKv8Dim);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (blk * kKv8Block + row0 + 16 * i < m) {
                float x[8];
                values(i, x);
                *reinterpret_cast<uint4*>(tail + (row0 + 16 * i) * kKv8Dim + chunk * 8) = pack_bf16x8(x);
            }
    }
}

}  // namespace minf

using namespace minf;

extern "C" int minf_kv8_store(
    const minf_kv8_cache* cache, const void* key, const void* value, const int64_t k_strides[3], const int64_t v_strides[3],
    int n_tokens, const int32_t* start, int start_all, const int32_t* counts, void* stream) {
    if (int rc = kv8_check(cache)) return rc;
    if (n_tokens && (!key || !value || !k_strides || !v_strides)) return fail(MINF_E_ARG, "null pointer argument");
    if (n_tokens < 0) return fail(MINF_E_ARG, "n_tokens must not be negative (got %d)", n_tokens);
    if (!start && (start_all < 0 || start_all > cache->capacity)) return fail(MINF_E_ARG, "start %d is outside the cache of %d tokens", start_all, cache->capacity);
    if (!start && !counts && n_tokens > cache->capacity - start_all)
        return fail(MINF_E_ARG, "%d tokens from position %d do not fit a cache of %d", n_tokens, start_all, cache->capacity);
    if (n_tokens == 0) return MINF_OK;
    StoreArgs a{};
    a.c = *cache;
    a.src[0] = static_cast<const __nv_bfloat16*>(key);
    a.src[1] = static_cast<const __nv_bfloat16*>(value);
    for (int i = 0; i < 3; ++i) {
        a.stride[0][i] = k_strides[i];
        a.stride[1][i] = v_strides[i];
        if (k_strides[i] % 8 || v_strides[i] % 8) return fail(MINF_E_ARG, "strides must be multiples of 8 elements");
    }
    if ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15) return fail(MINF_E_ARG, "keys and values must be 16-byte aligned");
    a.n_tokens = n_tokens;
    a.start = start;
    a.start_all = start_all;
    a.counts = counts;
    // the last position decides how many blocks can be touched: a start anywhere in its block, clipped by the capacity
    const int blocks = (int)min((long long)cache->capacity / kKv8Block, ((long long)n_tokens + 2 * kKv8Block - 2) / kKv8Block);
    dim3 grid(blocks, 2 * cache->heads, cache->batch);
    if (cache->format == MINF_KV8_E4M3)
        kv8_store_kernel<MINF_KV8_E4M3><<<grid, kStoreThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    else
        kv8_store_kernel<MINF_KV8_INT8><<<grid, kStoreThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    MINF_LAUNCH_OK("kv8_store_kernel");
    return MINF_OK;
}

extern "C" int minf_kv8_load(
    const minf_kv8_cache* cache, const int32_t* lengths, int length_all, const int32_t* first, int first_all, int count,
    void* k_out, void* v_out, void* stream) {
    if (int rc = kv8_check(cache)) return rc;
    if (count < 0 || count > (1 << 30)) return fail(MINF_E_ARG, "bad count %d", count);
    if (!lengths && (length_all < 0 || length_all > cache->capacity)) return fail(MINF_E_ARG, "length %d is outside the cache of %d tokens", length_all, cache->capacity);
    if (count == 0) return MINF_OK;
    if (!k_out || !v_out) return fail(MINF_E_ARG, "null pointer argument");
    if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) return fail(MINF_E_ARG, "outputs must be 16-byte aligned");
    LoadArgs a{};
    a.c = *cache;
    a.lengths = lengths;
    a.length_all = length_all;
    a.first = first;
    a.first_all = first_all;
    a.count = count;
    a.out[0] = static_cast<__nv_bfloat16*>(k_out);
    a.out[1] = static_cast<__nv_bfloat16*>(v_out);
    dim3 grid((count + kKv8Block - 1) / kKv8Block, 2 * cache->heads, cache->batch);
    if (cache->format == MINF_KV8_E4M3)
        kv8_load_kernel<MINF_KV8_E4M3><<<grid, kStoreThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    else
        kv8_load_kernel<MINF_KV8_INT8><<<grid, kStoreThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    MINF_LAUNCH_OK("kv8_load_kernel");
    return MINF_OK;
}

extern "C" int minf_kv8_evict(
    const minf_kv8_cache* src, const minf_kv8_cache* dst, const int32_t* lengths, int length_all, int max_length,
    const float* weights, const int64_t w_strides[2], int budget, int recent, int sink,
    int32_t* kept, float* weights_out, int32_t* lengths_out, void* stream) {
    if (int rc = kv8_check(src)) return rc;
    if (int rc = kv8_check(dst)) return rc;
    if (!weights || !w_strides || !kept || !weights_out || !lengths_out) return fail(MINF_E_ARG, "null pointer argument");
    if (src->format != dst->format || src->batch != dst->batch || src->heads != dst->heads)
        return fail(MINF_E_ARG, "the two caches must have one format, batch and head count");
    {
        auto overlap = [](const void* p, size_t np, const void* q, size_t nq) {
            const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
            return a < b + nq && b < a + np;
        };
        const size_t pairs = (size_t)src->batch * src->heads, tails = pairs * kKv8Block * kKv8Dim * 2;
        const void* from[6] = {src->k, src->v, src->k_scale, src->v_scale, src->k_tail, src->v_tail};
        const void* to[6] = {dst->k, dst->v, dst->k_scale, dst->v_scale, dst->k_tail, dst->v_tail};
        auto bytes = [&](const minf_kv8_cache* c, int i) {
            return i < 2 ? pairs * c->capacity * kKv8Dim : i < 4 ? pairs * (c->capacity / kKv8Block) * sizeof(float) : tails;
        };
        for (int i = 0; i < 6; ++i)
            for (int j = 0; j < 6; ++j)
                if (overlap(from[i], bytes(src, i), to[j], bytes(dst, j))) return fail(MINF_E_ARG, "eviction writes into another cache than it reads");
    }
    if (budget < 1 || recent < 0 || sink < 0 || (long long)recent + sink > budget)
        return fail(MINF_E_ARG, "budget %d must hold the %d first and %d last tokens", budget, sink, recent);
    if (budget > dst->capacity) return fail(MINF_E_ARG, "budget %d does not fit a cache of %d tokens", budget, dst->capacity);
    if (!lengths && (length_all < 0 || length_all > max_length)) return fail(MINF_E_ARG, "length %d is outside [0, max_length %d]", length_all, max_length);
    if (max_length < 0 || max_length > src->capacity) return fail(MINF_E_ARG, "max_length %d is outside the cache of %d tokens", max_length, src->capacity);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    SelectArgsKv8 a{};
    a.c = *src;
    a.lengths = lengths;
    a.length_all = length_all;
    a.max_length = max_length;
    a.weights = weights;
    a.w_stride[0] = w_strides[0];
    a.w_stride[1] = w_strides[1];
    a.budget = budget;
    a.recent = recent;
    a.sink = sink;
    a.kept = kept;
    // a CTA for every kSelectPart tokens, a power of two of them
    int parts = 1;
    while (parts < kSelectCluster && (long long)max_length > (long long)parts * kSelectPart) parts *= 2;
    a.cached = std::min(kSelectCached, (max_length / parts + 64) / 32 * 32);
    const size_t shared = (size_t)(kSelectWords + a.cached) * 4;
    static std::atomic<unsigned long long> allowed{0};
    MINF_CUDA_OK(allow_shared(kv8_select_kernel, (kSelectWords + kSelectCached) * 4, allowed));
    {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = parts;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(src->heads * parts, src->batch);
        cfg.blockDim = dim3(kSelectThreads);
        cfg.dynamicSmemBytes = shared;
        cfg.stream = s;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        MINF_CUDA_OK(cudaLaunchKernelEx(&cfg, kv8_select_kernel, a));
    }
    GatherArgs g{};
    g.src = *src;
    g.dst = *dst;
    g.lengths = lengths;
    g.length_all = length_all;
    g.max_length = max_length;
    g.weights = weights;
    g.w_stride[0] = w_strides[0];
    g.w_stride[1] = w_strides[1];
    g.budget = budget;
    g.kept = kept;
    g.weights_out = weights_out;
    g.lengths_out = lengths_out;
    dim3 grid(dst->capacity / kKv8Block, 2 * src->heads, src->batch);
    MINF_CUDA_OK(src->format == MINF_KV8_E4M3 ? launch_behind(kv8_gather_kernel<MINF_KV8_E4M3>, grid, kStoreThreads, 0, s, g)
                                              : launch_behind(kv8_gather_kernel<MINF_KV8_INT8>, grid, kStoreThreads, 0, s, g));
    return MINF_OK;
}
