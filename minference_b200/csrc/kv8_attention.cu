// Attention over an 8-bit key/value cache (layout: kv8.cuh): decoding steps of one or a few tokens, and longer ones.
//
// For a row (query head, query token) with logits l_t = sm_scale log2(e) s_K,t (q . c_K,t) over the tokens it sees,
//   out = sum_t 2^(l_t - lse) s_V,t c_V,t,    lse = log2 sum_t 2^l_t
// in one pass over the cache.  The running maximum M is that of l_t + log2 s_V,t, so the numerators
// P_t = 2^(l_t + log2 s_V,t - M) are at most 2^8 (M follows jumps beyond that only) and multiply the codes as they are; the
// denominator is the sum over blocks of (sum P_t) / s_V.  (All of it holds while the scales of the values of one head stay within
// 2^100 of each other, below which a block's numerators leave fp32, and the tail's values, which have no scale, below 2^104.)
//
// The products run on the tensor cores with the tokens as rows: S^T = K Q^T and O^T = V^T P^T, m16n8k16 in f16 with
// fp32 accumulation.  Eight query rows (a group of query heads that share a cache head, times the new tokens) fill the
// narrow side without padding to sixteen, and a code becomes an f16 value exactly.  Q is scaled by a power of two per
// row so that its bf16 values are f16 values (what is lost lies 2^-24 below the row's largest).  P is rounded to f16 with the
// headroom of kv8_attention.cuh: half a step of 2^-11 relative, below the bf16 rounding of the output, or 2^-32 of the largest;
// sums and outputs are accumulated in fp32.
// The tail (bf16) takes bf16 products, with P as a sum of two bf16 numbers.
//
// The tokens are split over CTAs and, inside one, over warps by units of 32.  Parts are joined by their log-sum-exps: short
// sequences' inside a cluster, others' in a second kernel, launched behind the first one's end.
//
// Bound: HBM.  Decoding steps of 4 rows per head read 131072 tokens of 8 heads in 45 us (5.9 TB/s; 51 us with the second
// kernel), 1048576 tokens in 310 us (6.9 TB/s), issue slots 43 % (int8: 53 %) and tensor pipe 18 % busy.  Up to 16 rows take
// 57 us, up to 24 75 us: there it is the chain of each warp (three warps a scheduler instead of two change nothing).
#include "kv8_attention.cuh"

#include <cooperative_groups.h>
#include <math_constants.h>

#include <algorithm>

#include "sm100_ptx.cuh"

namespace minf {

constexpr int kUnit = 32;                           // tokens a warp takes at a time: half a block
constexpr int kSlotBytes = kUnit * kKv8Dim;         // their keys or values
constexpr int kRingSlots = 3;
// Rows per cache head this kernel takes; more go to the wide one.  At 131072 tokens of 8 heads (e4m3, device time): 24 rows 76 us
// here and 85 us there, 32 rows (a fourth group, since removed) 97 and 90; four sequences of 16384: 32 rows 78 and 57.
constexpr int kNarrowRows = 24;
constexpr int kMaxCluster = 8;
// warps of a CTA: two CTAs fit an SM with 128 registers a thread for one group of rows, twice that for more
__host__ __device__ constexpr int narrow_warps(int nt) { return nt == 1 ? 8 : 4; }

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes are read once a call: they leave L2 before the logits and partial results that the second kernel reads.
__device__ __forceinline__ uint64_t stream_policy() {
    uint64_t p;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void cp_async_16_stream(uint32_t dst, const void* src, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Halves (f16, or bf16) that are infinite or NaN become zero; true if there were any.
template <bool BF16>
__device__ __forceinline__ bool drop_not_finite(uint32_t& x) {
    constexpr uint32_t m = BF16 ? 0x7f80u : 0x7c00u;
    const bool lo = (x & m) == m, hi = (x & (m << 16)) == (m << 16);
    if (lo) x &= 0xffff0000u;
    if (hi) x &= 0x0000ffffu;
    return lo || hi;
}

// What a warp carries along its tokens, for NT groups of eight rows: a lane holds columns 2c and 2c+1 of each group
// (c = lane % 4), and of the outputs dims 16g .. 16g+15 (g = lane / 4): o[nt][i] = {(dim 2i, col 2c), (2i, 2c+1),
// (2i+1, 2c), (2i+1, 2c+1)} of those.
template <int NT>
struct Rows {
    float o[NT][8][4];
    float m[NT][2];                 // running maximum of l + log2 s_V
    float l[NT][2];                 // this lane's part of the denominator, relative to m
    float mul[NT][2];               // logit of a unit of the accumulator, before the block's scale
};

// Logits of 16 * SUB tokens -> P, with the running statistics moved on.  s[j][nt][e]: token t0 + 16 j + tg (+ 8 for e = 2, 3),
// column 2c (+ 1 for odd e).  On return s holds P.  Where `masked`, a row sees the tokens below all_see + its own token's
// number only (columns behind the last row: anything, they are dropped).
template <int NT, int SUB, bool LOGITS>
__device__ __forceinline__ void softmax_step(const Kv8AttnArgs& a, Rows<NT>& R, float (&s)[SUB][NT][4], float k_scale, float v_scale,
                                             int t0, bool masked, int all_see, int end, size_t bh, int tg, int c) {
    const float lv = __log2f(v_scale), inv_v = __fdividef(kHeadroomOut, v_scale);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const float f0 = R.mul[nt][0] * k_scale, f1 = R.mul[nt][1] * k_scale;
        float mx0 = -CUDART_INF_F, mx1 = -CUDART_INF_F;
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            float* x = s[j][nt];
            x[0] *= f0;
            x[1] *= f1;
            x[2] *= f0;
            x[3] *= f1;
        }
        if (masked) {
            const int r = 8 * nt + 2 * c;
            const int lim0 = all_see + (a.n_q == 1 ? 0 : r % a.n_q), lim1 = all_see + (a.n_q == 1 ? 0 : (r + 1) % a.n_q);
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                float* x = s[j][nt];
                const int t = t0 + 16 * j + tg;
                if (t >= lim0) x[0] = -CUDART_INF_F;
                if (t >= lim1) x[1] = -CUDART_INF_F;
                if (t + 8 >= lim0) x[2] = -CUDART_INF_F;
                if (t + 8 >= lim1) x[3] = -CUDART_INF_F;
            }
        }
        if (LOGITS) {
            const int col = 8 * nt + 2 * c;
            if (col < a.pitch) {
                float* p = a.logits + ((long long)bh * a.tokens + t0 + tg) * a.pitch + col;
#pragma unroll
                for (int j = 0; j < SUB; ++j) {
                    const float* x = s[j][nt];
                    const int t = t0 + 16 * j + tg;
                    if (t < end) *reinterpret_cast<float2*>(p + 16 * j * a.pitch) = make_float2(x[0], x[1]);
                    if (t + 8 < end) *reinterpret_cast<float2*>(p + (16 * j + 8) * a.pitch) = make_float2(x[2], x[3]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            const float* x = s[j][nt];
            mx0 = fmaxf(mx0, fmaxf(x[0], x[2]));
            mx1 = fmaxf(mx1, fmaxf(x[1], x[3]));
        }
        // the reference is raised on a jump of more than 2^8: P stays below f16's largest, outputs are rarely rescaled, and the
        // lanes compare their maxima only then
        mx0 += lv;
        mx1 += lv;
        if (__any_sync(0xffffffffu, mx0 > R.m[nt][0] + 8.f || mx1 > R.m[nt][1] + 8.f)) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
                mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
            }
            const bool up0 = mx0 > R.m[nt][0] + 8.f, up1 = mx1 > R.m[nt][1] + 8.f;
            const float a0 = up0 ? fast_exp2(R.m[nt][0] - mx0) : 1.f, a1 = up1 ? fast_exp2(R.m[nt][1] - mx1) : 1.f;
            if (up0) R.m[nt][0] = mx0;
            if (up1) R.m[nt][1] = mx1;
            R.l[nt][0] *= a0;
            R.l[nt][1] *= a1;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                R.o[nt][i][0] *= a0;
                R.o[nt][i][1] *= a1;
                R.o[nt][i][2] *= a0;
                R.o[nt][i][3] *= a1;
            }
        }
        // nothing seen yet: -inf - 0
        const float d0 = lv + kHeadroom - (R.m[nt][0] == -CUDART_INF_F ? 0.f : R.m[nt][0]), d1 = lv + kHeadroom - (R.m[nt][1] == -CUDART_INF_F ? 0.f : R.m[nt][1]);
        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
            float* x = s[j][nt];
            x[0] = fast_exp2(x[0] + d0);
            x[1] = fast_exp2(x[1] + d1);
            x[2] = fast_exp2(x[2] + d0);
            x[3] = fast_exp2(x[3] + d1);
            sum0 += x[0] + x[2];
            sum1 += x[1] + x[3];
        }
        R.l[nt][0] = fmaf(sum0, inv_v, R.l[nt][0]);
        R.l[nt][1] = fmaf(sum1, inv_v, R.l[nt][1]);
    }
}

// How the narrow kernel's CTAs share the work of long sequences: the tokens of all sequences and heads are one row of units, (sequence, head,
// unit) in that order, and CTA i of N takes the units [U i / N, U (i + 1) / N).  Sequences of any lengths keep every CTA
// equally busy; where a CTA's share crosses into another head or sequence, it works on pieces one after the other.  The
// tail counts as a unit for each of the W warps.  Every CTA finds its place from the lengths by itself (a warp scans 32
// sequences at a time), so lengths may live on the device.
struct Place {
    int b, h, u, n;
};
template <int W>
__host__ __device__ constexpr int units_of(int n) {
    return n / kKv8Block * (kKv8Block / kUnit) + (n % kKv8Block ? W : 0);
}
__device__ __forceinline__ int clipped_length(const Kv8AttnArgs& a, int b) {
    const int n = a.lengths ? a.lengths[b] : a.length_all;
    return max(0, min(n, a.max_length));
}
struct Share {
    long long units;                // of all sequences and heads
    int ctas;                       // that get some: every warp of one a unit, as far as there are
    // of sequence `lane`, for batches of up to 32: tokens, units of a head, units of a head of it and those before
    int n, per, upto;
};
template <int W>
__device__ __forceinline__ Share share_of(const Kv8AttnArgs& a, bool report) {
    const int pairs = a.c.batch * a.c.heads, lane = threadIdx.x & 31;
    Share s{};
    bool same = true;               // sequences of one length
    if (!a.lengths) {
        s.units = (long long)pairs * units_of<W>(a.length_all);
    } else {
        int first = 0;
        for (int b0 = 0; b0 < a.c.batch; b0 += 32) {
            s.n = s.per = 0;
            const bool there = b0 + lane < a.c.batch;
            if (there) {
                const int n = a.lengths[b0 + lane];
                s.n = max(0, min(n, a.max_length));
                s.per = units_of<W>(s.n);
                if (report && threadIdx.x < 32 && n != s.n) atomicOr(a.c.status + MINF_ST_ERROR, MINF_ERR_KV8_RANGE);
            }
            if (b0 == 0) first = __shfl_sync(0xffffffffu, s.per, 0);
            same = same && (!there || s.per == first);
            s.upto = s.per;         // below 2^31: 32 sequences of at most 2^25 units and a tail
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, s.upto, o);
                if (lane >= o) s.upto += y;
            }
            s.units += __shfl_sync(0xffffffffu, s.upto, 31);
        }
        same = __all_sync(0xffffffffu, same);
        s.units *= a.c.heads;
    }
    s.ctas = a.splits;
    // a whole number of CTAs per head where that leaves few of them idle: then none works on two pieces, which costs it a new
    // start and a second joining
    if (same && pairs <= s.ctas && s.ctas / pairs * pairs * 10 >= s.ctas * 9) s.ctas = s.ctas / pairs * pairs;
    if (s.units < (long long)s.ctas * W) s.ctas = (int)((s.units + W - 1) / W);
    return s;
}
// x * y / z of non-negative numbers; 64-bit division takes a few hundred cycles, so it is left to products that need it
__device__ __forceinline__ long long mul_div(long long x, int y, long long z) {
    const long long p = x * y;
    return (p | z) >> 32 ? p / z : (long long)((unsigned)p / (unsigned)z);
}
// the CTA that has a unit
__device__ __forceinline__ long long owner_of(long long unit, long long units, int ctas) {
    const long long p = (unit + 1) * ctas - 1;
    return (p | units) >> 32 ? p / units : (long long)((unsigned)p / (unsigned)units);
}

template <int W>
__device__ __forceinline__ Place locate(const Kv8AttnArgs& a, const Share& share, long long at) {
    const int lane = threadIdx.x & 31;
    if (!a.lengths) {
        const int per = units_of<W>(a.length_all);
        const int bh = (int)mul_div(at, 1, per);
        return {bh / a.c.heads, bh % a.c.heads, (int)(at - (long long)bh * per), a.length_all};
    }
    for (int b0 = 0;; b0 += 32) {
        int n = share.n, per = share.per, upto = share.upto;
        if (a.c.batch > 32) {                       // the share has the last 32 only
            n = b0 + lane < a.c.batch ? clipped_length(a, b0 + lane) : 0;
            upto = per = units_of<W>(n);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
        }
        const unsigned here = __ballot_sync(0xffffffffu, at < (long long)upto * a.c.heads);
        if (here) {
            const int src = __ffs(here) - 1;
            const int nb = __shfl_sync(0xffffffffu, n, src), pb = __shfl_sync(0xffffffffu, per, src), ub = __shfl_sync(0xffffffffu, upto, src);
            const long long rest = at - (long long)(ub - pb) * a.c.heads;       // within the sequence's heads
            const int head = (int)mul_div(rest, 1, pb);
            return {b0 + src, head, (int)(rest - (long long)head * pb), nb};
        }
        if (b0 + 32 >= a.c.batch) return {0, 0, 0, 0};          // (not reached: `at` is below the total)
        at -= (long long)__shfl_sync(0xffffffffu, upto, 31) * a.c.heads;
    }
}
// units of a head of sequence b, and of all heads of the sequences before it
template <int W>
__device__ __forceinline__ void units_before(const Kv8AttnArgs& a, const Share& share, int b, int& per, long long& before) {
    if (!a.lengths) {
        per = units_of<W>(a.length_all);
        before = (long long)b * a.c.heads * per;
        return;
    }
    if (a.c.batch <= 32) {
        per = __shfl_sync(0xffffffffu, share.per, b);
        before = (long long)(__shfl_sync(0xffffffffu, share.upto, b) - per) * a.c.heads;
        return;
    }
    const int lane = threadIdx.x & 31;
    per = units_of<W>(clipped_length(a, b));
    before = 0;
    for (int b0 = 0; b0 < b; b0 += 32) {
        int x = b0 + lane < b ? units_of<W>(clipped_length(a, b0 + lane)) : 0;
#pragma unroll
        for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        before += x;
    }
    before *= a.c.heads;
}

template <int FMT, int NT, bool LOGITS>
__global__ void __launch_bounds__(narrow_warps(NT) * 32, 2) kv8_attention_kernel(const __grid_constant__ Kv8AttnArgs a) {
    constexpr int kAttnWarps = narrow_warps(NT), kAttnThreads = kAttnWarps * 32, kRingBytes = kAttnWarps * kRingSlots * kSlotBytes;
    constexpr int SUB = NT == 2 ? 2 : 1;            // sub-tiles of 16 tokens per softmax step: two hide latencies where registers allow
    constexpr int PARTS = kUnit / 16 / SUB;         // softmax steps of a unit
    constexpr bool kQShared = NT > 2;               // Q's fragments in shared memory (from there each is read once per sub-tile)
    extern __shared__ __align__(128) unsigned char ring_all[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    dependents_launch();
    Share share{};
    long long at = 0, stop = 1;                     // a cluster per head: one piece
    if (!a.cluster) {
        share = share_of<kAttnWarps>(a, blockIdx.x == 0);
        if ((int)blockIdx.x >= share.ctas) return;
        at = mul_div(share.units, blockIdx.x, share.ctas);
        stop = mul_div(share.units, blockIdx.x + 1, share.ctas);
    }
#pragma unroll 1
    while (at < stop) {                             // a piece: units of one sequence and head
    Place place;
    int rank = 0;
    if (a.cluster) {
        const int pair = blockIdx.x / a.cluster;
        rank = blockIdx.x % a.cluster;
        place.b = pair / a.c.heads;
        place.h = pair % a.c.heads;
        place.n = kv8_length(a.lengths, a.length_all, place.b, a.max_length, a.c.status);
        place.u = units_of<kAttnWarps>(place.n) * rank / a.cluster;
    } else {
        place = locate<kAttnWarps>(a, share, at);
    }
    const int h = place.h, b = place.b, n = place.n;
    const size_t bh = (size_t)b * a.c.heads + h;
    const int full = n / kKv8Block;                 // complete blocks
    const int full_u = full * (kKv8Block / kUnit), units = units_of<kAttnWarps>(n);
    const int x_lo = place.u, x_hi = a.cluster ? units * (rank + 1) / a.cluster : (int)min((long long)units, x_lo + (stop - at));
    const int u_lo = min(full_u, x_lo), u_hi = min(full_u, x_hi);
    const bool takes_tail = x_hi == units;          // the tail's units: its last one's piece takes all of it
    const bool whole = a.cluster == 1 || (!a.cluster && x_lo == 0 && x_hi == units);     // nothing to join: the output is written here
    const size_t piece = blockIdx.x + bh;           // pieces are numbered so: both grow along the units, one of them at each new piece
    at = a.cluster ? stop : at + (x_hi - x_lo);
    if (takes_tail && n % kKv8Block) {              // the tail is wanted at the end: on its way to L2 from here
        const char* kt = reinterpret_cast<const char*>(static_cast<const __nv_bfloat16*>(a.c.k_tail) + bh * kKv8Block * kKv8Dim);
        const char* vt = reinterpret_cast<const char*>(static_cast<const __nv_bfloat16*>(a.c.v_tail) + bh * kKv8Block * kKv8Dim);
        for (int i = threadIdx.x * 128; i < kKv8Block * kKv8Dim * 2; i += kAttnThreads * 128) {
            asm volatile("prefetch.global.L2 [%0];" ::"l"(kt + i));
            asm volatile("prefetch.global.L2 [%0];" ::"l"(vt + i));
        }
    }
    const int all_see = n - a.n_q + 1;              // tokens below this are seen by every row

    // The warp's own ring of three slots of 4 KB: keys of a unit, values of it, keys of its next unit, ...; two copies
    // are in flight while the third is used.  16-byte chunk ch of row r lies at ch ^ (r & 7).
    unsigned char* const ring = ring_all + warp * (kRingSlots * kSlotBytes);
    const uint32_t ring_u = smem_u32(ring);
    const uint32_t put0 = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4), put1 = (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3) + 4)) << 4);
    const uint64_t stream = stream_policy();
    auto fetch = [&](int slot, const uint8_t* src) {
        src += lane * 16;
        const uint32_t dst = ring_u + slot * kSlotBytes;
#pragma unroll
        for (int i = 0; i < kSlotBytes / 512; ++i) cp_async_16_stream(dst + 512 * i + ((i & 1) ? put1 : put0), src + 512 * i, stream);
    };
    const float* ks = a.c.k_scale + bh * (a.c.capacity / kKv8Block);
    const float* vs = a.c.v_scale + bh * (a.c.capacity / kKv8Block);
    const size_t first = (bh * (a.c.capacity / kUnit) + u_lo + warp) * kSlotBytes;
    const uint8_t* next_k = static_cast<const uint8_t*>(a.c.k) + first;
    const uint8_t* next_v = static_cast<const uint8_t*>(a.c.v) + first;
    float k_scale = 1.f, v_scale = 1.f;
    auto scale_at = [](int u) { return u / (kKv8Block / kUnit); };
    if (u_lo + warp < u_hi) {
        fetch(0, next_k);
        cp_async_commit();
        fetch(1, next_v);
        k_scale = ks[scale_at(u_lo + warp)];
        v_scale = vs[scale_at(u_lo + warp)];
    } else {
        cp_async_commit();
    }
    cp_async_commit();

    // Q^T fragments: column g of group nt, dims of step s: 64 (s / 4) + 16 c + 4 (s % 4) + {0, 1 | 2, 3}.  Where they are
    // shared, warp nt makes those of group nt.
    Rows<NT> R;
    uint32_t qf[kQShared ? 1 : NT][8][2];
    uint2* const q_sm = reinterpret_cast<uint2*>(ring_all + kRingBytes);        // [nt][step][lane]
    float* const unit_sm = reinterpret_cast<float*>(ring_all + kRingBytes + NT * 2048);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float unit = 1.f;                           // power of two the row was divided by
        if (!kQShared || warp == nt) {
            const int r = 8 * nt + g;
            const uint4* q = nullptr;
            if (r < a.rows) {
                const int hq = h * a.group + (a.n_q == 1 ? r : r / a.n_q), t = a.n_q == 1 ? 0 : r % a.n_q;
                q = reinterpret_cast<const uint4*>(a.q + b * a.qs[0] + (long long)hq * a.qs[1] + (long long)t * a.qs[2]);
            }
            float top = 0.f;
            float x[4][8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {           // eight dims from 64 (i / 2) + 16 c + 8 (i % 2) on; zeros behind the last row
                bf16x8_to_values(q ? q[8 * (i >> 1) + 2 * c + (i & 1)] : make_uint4(0u, 0u, 0u, 0u), x[i]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float m = fabsf(x[i][e]);
                    if (m < CUDART_INF_F) top = fmaxf(top, m);
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            int e = 0;
            if (top > 0.f) frexpf(top, &e);         // top < 2^e: scaled to below 2^8, so that the smallest products count too
            e = max(e - 8, -126);
            const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
            unit = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                const float* v = &x[st >> 1][4 * (st & 1)];
                const uint32_t b0 = pack_half2(v[0] * inv, v[1] * inv), b1 = pack_half2(v[2] * inv, v[3] * inv);
                if constexpr (kQShared) {
                    q_sm[(nt * 8 + st) * 32 + lane] = make_uint2(b0, b1);
                } else {
                    qf[nt][st][0] = b0;
                    qf[nt][st][1] = b1;
                }
            }
            if (kQShared && c == 0) unit_sm[8 * nt + g] = unit;
        }
        if constexpr (!kQShared) {
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) R.mul[nt][cc] = a.scale_log2 * __shfl_sync(0xffffffffu, unit, 4 * (2 * c + cc));
        }
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
            R.m[nt][cc] = -CUDART_INF_F;
            R.l[nt][cc] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) R.o[nt][i][k] = 0.f;
    }
    if constexpr (kQShared) {
        static_assert(NT <= kAttnWarps, "a warp for each group");
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) R.mul[nt][cc] = a.scale_log2 * unit_sm[8 * nt + 2 * c + cc];
    }
    auto q_frag = [&](int nt, int st) {
        if constexpr (kQShared) return q_sm[(nt * 8 + st) * 32 + lane];
        else return make_uint2(qf[nt][st][0], qf[nt][st][1]);
    };

    // Row i of the eight of a fragment is token perm(i): with it, and the chunks' places in the ring, the eight lanes of a
    // quarter of a shared-memory access touch all 32 banks, for the keys' rows and for the values' alike.
    const int pg = (g & 1) ? (g - 1) ^ 5 : g;       // perm(g)
    const int pa = 2 * c, pb = (2 * c) ^ 5;         // perm(2c), perm(2c + 1)
    bool bad = false;                               // values left out of the products, see below

    constexpr size_t kHop = (size_t)kAttnWarps * kSlotBytes;
    int slot = 0;
    for (int u = u_lo + warp; u < u_hi; u += kAttnWarps) {
        const bool more = u + kAttnWarps < u_hi;
        const bool masked = (u + 1) * kUnit > all_see;
        const float ksc = k_scale, vsc = v_scale;
        next_k += kHop;
        next_v += kHop;
        const int slot_v = slot == 2 ? 0 : slot + 1, slot_n = slot_v == 2 ? 0 : slot_v + 1;
        if (more) {
            fetch(slot_n, next_k);
            k_scale = ks[scale_at(u + kAttnWarps)];
            v_scale = vs[scale_at(u + kAttnWarps)];
        }
        cp_async_commit();
        cp_async_wait<2>();
        __syncwarp();
        const unsigned char* kb = ring + slot * kSlotBytes;
        const unsigned char* vb = ring + slot_v * kSlotBytes;
        bool v_here = false;
#pragma unroll 1
        for (int part = 0; part < PARTS; ++part) {
            const int t0 = u * kUnit + part * SUB * 16;
            float s[SUB][NT][4];
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                const unsigned char* p = kb + (part * SUB * 16 + 16 * j + pg) * kKv8Dim;       // rows pg and pg + 8: the same r & 7
                const uint4 k00 = *reinterpret_cast<const uint4*>(p + ((c ^ pg) << 4));
                const uint4 k01 = *reinterpret_cast<const uint4*>(p + (((c + 4) ^ pg) << 4));
                const uint4 k10 = *reinterpret_cast<const uint4*>(p + 8 * kKv8Dim + ((c ^ pg) << 4));
                const uint4 k11 = *reinterpret_cast<const uint4*>(p + 8 * kKv8Dim + (((c + 4) ^ pg) << 4));
                const uint32_t r0[8] = {k00.x, k00.y, k00.z, k00.w, k01.x, k01.y, k01.z, k01.w};
                const uint32_t r1[8] = {k10.x, k10.y, k10.z, k10.w, k11.x, k11.y, k11.z, k11.w};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j][nt][e] = 0.f;
#pragma unroll
                for (int st = 0; st < 8; ++st) {
                    uint32_t a0, a1, a2, a3;
                    codes_to_half<FMT>(r0[st], a0, a2);
                    codes_to_half<FMT>(r1[st], a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint2 q = q_frag(nt, st);
                        mma_f16(s[j][nt], a0, a1, a2, a3, q.x, q.y);
                    }
                }
            }
            softmax_step<NT, SUB, LOGITS>(a, R, s, ksc, vsc, t0, masked, all_see, n, bh, pg, c);
            if (!v_here) {
                cp_async_wait<1>();
                __syncwarp();
                v_here = true;
            }
#pragma unroll
            for (int j = 0; j < SUB; ++j) {
                uint32_t b0[NT], b1[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    b0[nt] = transpose8x8(pack_half2(s[j][nt][0], s[j][nt][1]));
                    b1[nt] = transpose8x8(pack_half2(s[j][nt][2], s[j][nt][3]));
                }
                // A fragments of V^T: two tokens in the halves of a register, rows g and g + 8 are dims 16g+2i, 16g+2i+1
                const unsigned char* p = vb + (part * SUB * 16 + 16 * j) * kKv8Dim;
                const uint4 x0 = *reinterpret_cast<const uint4*>(p + pa * kKv8Dim + ((g ^ pa) << 4));
                const uint4 y0 = *reinterpret_cast<const uint4*>(p + pb * kKv8Dim + ((g ^ pb) << 4));
                const uint4 x1 = *reinterpret_cast<const uint4*>(p + (pa + 8) * kKv8Dim + ((g ^ pa) << 4));
                const uint4 y1 = *reinterpret_cast<const uint4*>(p + (pb + 8) * kKv8Dim + ((g ^ pb) << 4));
                const uint32_t xs0[4] = {x0.x, x0.y, x0.z, x0.w}, ys0[4] = {y0.x, y0.y, y0.z, y0.w};
                const uint32_t xs1[4] = {x1.x, x1.y, x1.z, x1.w}, ys1[4] = {y1.x, y1.y, y1.z, y1.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t sel = (i & 1) ? 0x7362 : 0x5140;
                    uint32_t v0, v1, v2, v3;
                    codes_to_half<FMT>(__byte_perm(xs0[i >> 1], ys0[i >> 1], sel), v0, v1);
                    codes_to_half<FMT>(__byte_perm(xs1[i >> 1], ys1[i >> 1], sel), v2, v3);
                    if (FMT == MINF_KV8_E4M3 && masked) {
                        bad |= drop_not_finite<false>(v0);
                        bad |= drop_not_finite<false>(v1);
                        bad |= drop_not_finite<false>(v2);
                        bad |= drop_not_finite<false>(v3);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_f16(R.o[nt][i], v0, v1, v2, v3, b0[nt], b1[nt]);
                }
            }
        }
        __syncwarp();
        // both slots are free: the values of the next unit take the one the keys were in
        if (more) fetch(slot, next_v);
        cp_async_commit();
        slot = slot_n;
    }

    // the tail: four warps take 16 of its tokens each
    const int t0 = full * kKv8Block + 16 * warp;
    if (takes_tail && warp < 4 && t0 < n) {
        const __nv_bfloat16* kt = static_cast<const __nv_bfloat16*>(a.c.k_tail) + (bh * kKv8Block + 16 * warp) * kKv8Dim;
        const __nv_bfloat16* vt = static_cast<const __nv_bfloat16*>(a.c.v_tail) + (bh * kKv8Block + 16 * warp) * kKv8Dim;
        float s[1][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0][nt][e] = 0.f;
        auto to_bf16 = [](uint32_t x) {             // (eight bits of them at most: exact, but for what f16 has lost already)
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
            return pack_bf16x2(f.x, f.y);
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) {               // 16 dims of a lane quad: two steps
            const int d = 64 * (i >> 1) + 16 * c + 8 * (i & 1);
            const uint4 x = *reinterpret_cast<const uint4*>(kt + g * kKv8Dim + d), y = *reinterpret_cast<const uint4*>(kt + (g + 8) * kKv8Dim + d);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const uint2 q0 = q_frag(nt, 2 * i), q1 = q_frag(nt, 2 * i + 1);
                mma_bf16(s[0][nt], x.x, y.x, x.y, y.y, to_bf16(q0.x), to_bf16(q0.y));
                mma_bf16(s[0][nt], x.z, y.z, x.w, y.w, to_bf16(q1.x), to_bf16(q1.y));
            }
        }
        // tokens behind the last one must not count: no row sees them (all_see + n_q - 1 = n)
        softmax_step<NT, 1, LOGITS>(a, R, s, 1.f, 1.f, t0, true, all_see, n, bh, g, c);
        uint32_t h0[NT], h1[NT], e0[NT], e1[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float* x = s[0][nt];
            h0[nt] = pack_bf16x2(x[0], x[1]);
            h1[nt] = pack_bf16x2(x[2], x[3]);
            e0[nt] = transpose8x8(pack_bf16x2(x[0] - __uint_as_float(h0[nt] << 16), x[1] - __uint_as_float(h0[nt] & 0xffff0000u)));
            e1[nt] = transpose8x8(pack_bf16x2(x[2] - __uint_as_float(h1[nt] << 16), x[3] - __uint_as_float(h1[nt] & 0xffff0000u)));
            h0[nt] = transpose8x8(h0[nt]);
            h1[nt] = transpose8x8(h1[nt]);
        }
#pragma unroll
        for (int w = 0; w < 2; ++w) {               // eight dims of four tokens
            uint32_t xs[2][4], ys[2][4];
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
                const int r = 2 * c + 8 * hf;
                const __nv_bfloat16* p = vt + r * kKv8Dim + 16 * g + 8 * w;
                uint4 x = *reinterpret_cast<const uint4*>(p), y = *reinterpret_cast<const uint4*>(p + kKv8Dim);
                if (t0 + r >= n) x = make_uint4(0u, 0u, 0u, 0u);        // rows behind the last token hold anything
                if (t0 + r + 1 >= n) y = make_uint4(0u, 0u, 0u, 0u);
                xs[hf][0] = x.x; xs[hf][1] = x.y; xs[hf][2] = x.z; xs[hf][3] = x.w;
                ys[hf][0] = y.x; ys[hf][1] = y.y; ys[hf][2] = y.z; ys[hf][3] = y.w;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t v0 = __byte_perm(xs[0][k], ys[0][k], 0x5410), v1 = __byte_perm(xs[0][k], ys[0][k], 0x7632);
                uint32_t v2 = __byte_perm(xs[1][k], ys[1][k], 0x5410), v3 = __byte_perm(xs[1][k], ys[1][k], 0x7632);
                bad |= drop_not_finite<true>(v0);
                bad |= drop_not_finite<true>(v1);
                bad |= drop_not_finite<true>(v2);
                bad |= drop_not_finite<true>(v3);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma_bf16(R.o[nt][4 * w + k], v0, v1, v2, v3, h0[nt], h1[nt]);
                    mma_bf16(R.o[nt][4 * w + k], v0, v1, v2, v3, e0[nt], e1[nt]);
                }
            }
        }
    }

    // Join the warps, eight rows at a time.  In units that some row does not see to their end and in the tail, values that
    // are infinite or NaN were left out of the products (zero times them would not be zero) and are added here to the rows that see them.
    const bool any_bad = __syncthreads_or(bad);     // (and the rings are read out)
    constexpr int kRows = 8 * NT;
    float (*sm_o)[kRows][kKv8Dim] = reinterpret_cast<float (*)[kRows][kKv8Dim]>(ring_all);
    static_assert(kAttnWarps * kRows * kKv8Dim * sizeof(float) <= kRingBytes, "the warps' outputs fit the rings");
    __shared__ float2 sm_ml[kAttnWarps][kRows];     // maximum and denominator; then the warp's weight
    __shared__ float sm_lse[kRows];                 // of a cluster's part
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
            float l = R.l[nt][cc];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const int r = 8 * nt + 2 * c + cc;
            if (g == 0) sm_ml[warp][r] = make_float2(R.m[nt][cc], l);
            float* dst = &sm_o[warp][r][16 * g];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(dst + 4 * i) = make_float4(R.o[nt][2 * i][cc], R.o[nt][2 * i][2 + cc], R.o[nt][2 * i + 1][cc], R.o[nt][2 * i + 1][2 + cc]);
        }
    __syncthreads();
    if (threadIdx.x < kRows) {                      // a row's log-sum-exp, and what each warp's output counts for in it
        const int r = threadIdx.x;
        float lse[kAttnWarps], l[kAttnWarps], top = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
            const float2 x = sm_ml[w][r];
            l[w] = x.y;
            lse[w] = x.y == 0.f ? -CUDART_INF_F : x.x == -CUDART_INF_F ? x.y : x.x + log2f(x.y);
            top = fmaxf(top, lse[w]);
        }
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
            lse[w] = lse[w] == -CUDART_INF_F ? 0.f : exp2f(lse[w] - top);
            sum += lse[w];
        }
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) sm_ml[w][r].x = lse[w] == 0.f ? 0.f : lse[w] * kHeadroomOut / (sum * l[w]);
        const float all = sum == 0.f ? -CUDART_INF_F : top + log2f(sum);
        sm_lse[r] = all;
        if (r < a.rows) {
            if (!a.cluster) a.part_lse[piece * a.rows + r] = all;
            else if (whole && a.logits) a.part_lse[bh * a.rows + r] = all;
            if (whole && a.lse) {
                const int hq = h * a.group + r / a.n_q;
                a.lse[((size_t)b * a.c.heads * a.group + hq) * a.n_q + r % a.n_q] = all;
            }
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < kRows * 32; i += kAttnThreads) {
        const int r = i >> 5, d = (i & 31) * 4;
        if (r >= a.rows) break;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) {
            const float f = sm_ml[w][r].x;
            if (f == 0.f) continue;                 // (its output may be anything times zero)
            const float4 x = *reinterpret_cast<const float4*>(&sm_o[w][r][d]);
            acc[0] = fmaf(f, x.x, acc[0]);
            acc[1] = fmaf(f, x.y, acc[1]);
            acc[2] = fmaf(f, x.z, acc[2]);
            acc[3] = fmaf(f, x.w, acc[3]);
        }
        if (any_bad) {
            const int lo = max(u_lo * kUnit, min(max(all_see, 0) / kUnit * kUnit, full * kKv8Block)), lim = all_see + r % a.n_q;
            const int hi = min(takes_tail ? n : u_hi * kUnit, lim);
            for (int t = lo; t < hi; ++t)
                for (int k = 0; k < 4; ++k) {
                    float v = 0.f;
                    if (t >= full * kKv8Block)
                        v = __bfloat162float(static_cast<const __nv_bfloat16*>(a.c.v_tail)[(bh * kKv8Block + t % kKv8Block) * kKv8Dim + d + k]);
                    else if (FMT == MINF_KV8_E4M3 && (static_cast<const uint8_t*>(a.c.v)[(bh * a.c.capacity + t) * kKv8Dim + d + k] & 0x7f) == 0x7f)
                        v = CUDART_NAN_F;
                    if (!(fabsf(v) < CUDART_INF_F)) acc[k] += v;
                }
        }
        if (a.cluster > 1) {
            *reinterpret_cast<float4*>(&sm_o[0][r][d]) = make_float4(acc[0], acc[1], acc[2], acc[3]);     // (read by this thread alone)
        } else if (!whole) {
            *reinterpret_cast<float4*>(a.part_o + (piece * a.rows + r) * kKv8Dim + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        } else {
            const int hq = h * a.group + (a.n_q == 1 ? r : r / a.n_q), t = a.n_q == 1 ? 0 : r % a.n_q;
            __nv_bfloat16* o = a.o + b * a.os[0] + hq * a.os[1] + t * a.os[2] + d;
            *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
        }
    }
    if (a.cluster > 1) {
        // the parts of the cluster joined out of its CTAs' shared memories, each CTA some of the rows
        namespace cg = cooperative_groups;
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        for (int i = rank * kAttnThreads + threadIdx.x; i < a.rows * 32; i += a.cluster * kAttnThreads) {
            const int r = i >> 5, d = (i & 31) * 4;
            float e[kMaxCluster], top = -CUDART_INF_F, sum = 0.f;
            float4 x[kMaxCluster];
#pragma unroll
            for (int k = 0; k < kMaxCluster; ++k) {
                const int from = min(k, a.cluster - 1);
                e[k] = *cluster.map_shared_rank(&sm_lse[r], from);
                x[k] = *reinterpret_cast<const float4*>(cluster.map_shared_rank(&sm_o[0][r][d], from));
                if (k >= a.cluster) e[k] = -CUDART_INF_F;
                top = fmaxf(top, e[k]);
            }
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            const float ref = top == -CUDART_INF_F ? 0.f : top;
#pragma unroll
            for (int k = 0; k < kMaxCluster; ++k) {
                if (k >= a.cluster) break;
                const float f = exp2f(e[k] - ref);          // (a part that saw nothing holds zeros; NaN goes through)
                sum += f;
                acc.x = fmaf(f, x[k].x, acc.x);
                acc.y = fmaf(f, x[k].y, acc.y);
                acc.z = fmaf(f, x[k].z, acc.z);
                acc.w = fmaf(f, x[k].w, acc.w);
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int hq = h * a.group + (a.n_q == 1 ? r : r / a.n_q), t = a.n_q == 1 ? 0 : r % a.n_q;
            __nv_bfloat16* o = a.o + b * a.os[0] + hq * a.os[1] + t * a.os[2] + d;
            *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
            if (d == 0) {
                const float all = sum == 0.f ? -CUDART_INF_F : top + log2f(sum);
                if (a.logits) a.part_lse[bh * a.rows + r] = all;
                if (a.lse) a.lse[((size_t)b * a.c.heads * a.group + hq) * a.n_q + t] = all;
            }
        }
        cluster.sync();                             // the others read this CTA's part
    }
    __syncthreads();                                // before the next piece's copies
    }
}

// Loads that stay in their order before their uses, several in flight: the compiler may move plain ones to their uses.
__device__ __forceinline__ float load_now(const float* p) {
    float x;
    asm volatile("ld.global.f32 %0, [%1];" : "=f"(x) : "l"(p) : "memory");
    return x;
}
__device__ __forceinline__ float4 load_now4(const float* p) {
    float4 x;
    asm volatile("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "l"(p) : "memory");
    return x;
}

// Parts of a row: `count` of them, the first at row `base` of part_o / part_lse, `step` rows apart.
struct Parts {
    size_t base, step;
    int count;
};
template <int W>
__device__ __forceinline__ Parts parts_of(const Kv8AttnArgs& a, size_t bh, int r) {
    if constexpr (W == 0) {                         // wide kernel: a fixed number of splits
        return {(bh * a.rows + r) * a.splits, 1, a.splits};
    } else {
        const int b = (int)(bh / a.c.heads), h = (int)(bh % a.c.heads);
        if (a.cluster) return {bh * a.rows + r, (size_t)a.rows, 1};    // (its log-sum-exp, for the weights)
        const Share share = share_of<W>(a, false);
        const long long all = share.units;
        const int ctas = share.ctas;
        int per;
        long long start;
        units_before<W>(a, share, b, per, start);
        if (per == 0) return {0, 0, 0};
        start += (long long)h * per;
        const long long lo = owner_of(start, all, ctas), hi = owner_of(start + per - 1, all, ctas);
        return {((size_t)lo + bh) * a.rows + r, (size_t)a.rows, (int)(hi - lo + 1)};
    }
}

// The parts of one row joined and written: `WARPS` warps of the CTA take every WARPS-th part, a lane four dims.
template <int WARPS>
__device__ __forceinline__ void join_row(const Kv8AttnArgs& a, const Parts& p, size_t row, int warp, int lane, float4 (*sm)[32], float* sm_sum) {
    float top = -CUDART_INF_F;
    for (int k = lane; k < p.count; k += 32) top = fmaxf(top, a.part_lse[p.base + k * p.step]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const float ref = top == -CUDART_INF_F ? 0.f : top;
    for (int k0 = warp; k0 < p.count; k0 += 4 * WARPS) {
        float e[4];
        float4 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {               // (behind the last part: that one again, for nothing)
            const size_t at = p.base + min(k0 + u * WARPS, p.count - 1) * p.step;
            e[u] = load_now(a.part_lse + at);
            x[u] = load_now4(a.part_o + at * kKv8Dim + 4 * lane);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float f = k0 + u * WARPS < p.count ? exp2f(e[u] - ref) : 0.f;        // (a part that saw nothing holds zeros)
            sum += f;
            acc.x = fmaf(f, x[u].x, acc.x);
            acc.y = fmaf(f, x[u].y, acc.y);
            acc.z = fmaf(f, x[u].z, acc.z);
            acc.w = fmaf(f, x[u].w, acc.w);
        }
    }
    if constexpr (WARPS > 1) {
        sm[warp][lane] = acc;
        if (lane == 0) sm_sum[warp] = sum;
        __syncthreads();
        if (warp) return;
        sum = 0.f;
        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float4 x = sm[w][lane];
            sum += sm_sum[w];
            acc.x += x.x;
            acc.y += x.y;
            acc.z += x.z;
            acc.w += x.w;
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int bh = (int)(row / a.rows), r = (int)(row % a.rows), b = bh / a.c.heads, h = bh % a.c.heads;
    const int hq = h * a.group + r / a.n_q, t = r % a.n_q;
    __nv_bfloat16* o = a.o + b * a.os[0] + hq * a.os[1] + t * a.os[2] + 4 * lane;
    *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    if (lane == 0) {
        const float e = sum == 0.f ? -CUDART_INF_F : top + log2f(sum);
        if (a.lse) a.lse[((size_t)b * a.c.heads * a.group + hq) * a.n_q + t] = e;
        if (a.row_lse) a.row_lse[row] = e;
    }
}

constexpr int kFinishThreads = 256;
constexpr int kFinishTokens = 1024;                 // tokens that a CTA sums weights of at a time
constexpr int kFinishCtas = 8 * kSMs;               // CTAs of that kind worth starting: resident at once, each with some microseconds of start

// Weights of tokens [t0, t0 + kFinishTokens) of a head: the probabilities of its rows, summed in their order.  A thread has
// four tokens, whose logits it reads together.
// (no condition in it: one per element kept the loads from being in flight together, sixteen times the time)
__device__ __forceinline__ float weight_of(float logit, float lse) { return fast_exp2(logit - lse); }
// a row that sees nothing has logits of -inf: 2^(-inf - 0) = 0
__device__ __forceinline__ float for_weights(float lse) { return lse == -CUDART_INF_F ? 0.f : lse; }
__device__ __forceinline__ void sum_weights(const Kv8AttnArgs& a, int b, int h, int n, int t0, const float* row_lse) {
    constexpr int kEach = kFinishTokens / kFinishThreads;
    const size_t bh = (size_t)b * a.c.heads + h;
    const float* x = a.logits + ((long long)bh * a.tokens + t0 + threadIdx.x) * a.pitch;
    const float* add = a.add_to ? a.add_to + b * a.as[0] + h * a.as[1] + t0 + threadIdx.x : nullptr;
    const int left = n - t0 - (int)threadIdx.x;     // token k of this thread: k * kFinishThreads < left
    if (left <= 0) return;
    // behind the last token: an earlier one again, dropped at the end
    long long row[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) row[k] = (long long)(k * kFinishThreads < left ? k : 0) * kFinishThreads;
    float was[kEach], sum[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        was[k] = add ? load_now(add + row[k]) : 0.f;
        sum[k] = 0.f;
    }
    int r = 0;
    for (; r + 4 <= a.pitch; r += 4) {              // (a pitch of 2, or a multiple of 4)
        float4 l[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            l[k] = load_now4(x + row[k] * a.pitch + r);
        // columns behind the last row hold anything, NaN too: their finished terms are dropped
        const bool r1 = r + 1 < a.rows, r2 = r + 2 < a.rows, r3 = r + 3 < a.rows;
        const float e0 = row_lse[r], e1 = r1 ? row_lse[r + 1] : 0.f, e2 = r2 ? row_lse[r + 2] : 0.f, e3 = r3 ? row_lse[r + 3] : 0.f;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const float w1 = weight_of(l[k].y, e1), w2 = weight_of(l[k].z, e2), w3 = weight_of(l[k].w, e3);
            sum[k] += weight_of(l[k].x, e0);
            sum[k] += r1 ? w1 : 0.f;
            sum[k] += r2 ? w2 : 0.f;
            sum[k] += r3 ? w3 : 0.f;
        }
    }
    if (a.pitch == 2) {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const float2 l = *reinterpret_cast<const float2*>(x + row[k] * 2);
            sum[k] += weight_of(l.x, row_lse[0]);
            if (a.rows > 1) sum[k] += weight_of(l.y, row_lse[1]);
        }
    }
    float* w = a.weights + b * a.ws[0] + h * a.ws[1] + t0 + threadIdx.x;
#pragma unroll
    for (int k = 0; k < kEach; ++k)
        if (k * kFinishThreads < left) w[k * kFinishThreads] = was[k] + sum[k];
}

// The first CTAs join the parts of a row each (narrow kernel: up to a few dozen parts, eight warps) or of eight rows (wide
// kernel).  The others (narrow kernel) sum the weights, for which they join the log-sum-exps of their head's rows themselves: no
// second wait.  Behind the attention of 131072 tokens it takes 4-5 us; with the weights of 262144 tokens and 28 query heads,
// whose 34 MB of logits come out of L2, 13 us.
template <int W>
__global__ void __launch_bounds__(kFinishThreads) kv8_finish_kernel(const __grid_constant__ Kv8AttnArgs a) {
    __shared__ float4 sm[8][32];
    __shared__ float sm_sum[8];
    __shared__ float sm_lse[kNarrowRows];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const size_t rows = (size_t)a.c.batch * a.c.heads * a.rows;
    dependents_launch();
    if (blockIdx.x >= rows) {
        if constexpr (W > 0) {
            const int chunks = (int)((a.tokens + a.chunk - 1) / a.chunk);
            const int i = (int)(blockIdx.x - rows), chunk = i % chunks;
            const size_t bh = i / chunks;
            const int b = (int)(bh / a.c.heads), h = (int)(bh % a.c.heads);
            const int n = clipped_length(a, b);
            const Parts p = parts_of<W>(a, bh, 0);
            dependents_wait();
            if ((long long)chunk * a.chunk >= n) return;
            for (int r = warp; r < a.rows; r += 8) {
                float top = -CUDART_INF_F, sum = 0.f;
                for (int k = lane; k < p.count; k += 32) top = fmaxf(top, a.part_lse[p.base + r + k * p.step]);
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                for (int k = lane; k < p.count; k += 32) {
                    const float e = a.part_lse[p.base + r + k * p.step];
                    sum += e == -CUDART_INF_F ? 0.f : exp2f(e - top);
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (lane == 0) sm_lse[r] = for_weights(sum == 0.f ? -CUDART_INF_F : top + log2f(sum));
            }
            __syncthreads();
            for (int t0 = chunk * a.chunk; t0 < min((long long)n, (chunk + 1ll) * a.chunk); t0 += kFinishTokens) sum_weights(a, b, h, n, t0, sm_lse);
        }
        return;
    }
    if constexpr (W == 0) {                         // the wide kernel's few splits: a warp per row
        const size_t row = (size_t)blockIdx.x * 8 + warp;
        dependents_wait();
        if (row < rows) join_row<1>(a, {row * a.splits, 1, a.splits}, row, 0, lane, nullptr, nullptr);
        return;
    }
    const size_t bh = blockIdx.x / a.rows;
    const int r = (int)(blockIdx.x % a.rows);
    const Parts p = parts_of<W>(a, bh, r);
    dependents_wait();
    if (W > 0 && p.count == 1) return;              // the attention kernel wrote this row itself
    join_row<8>(a, p, bh * a.rows + r, warp, lane, sm, sm_sum);
}

// Weights after the wide kernel, whose rows' log-sum-exps are joined by then: a warp has eight tokens and takes 128 rows of
// them at a time through shared memory, four a lane.  (With plain loads, which the compiler put next to their uses, 448 rows of
// 8000 tokens took 104 us instead of 20.)
constexpr int kWideTokensWarp = 8, kWeightThreads = 128, kWideTokens = kWideTokensWarp * kWeightThreads / 32;
__global__ void __launch_bounds__(kWeightThreads) kv8_weights_kernel(const __grid_constant__ Kv8AttnArgs a) {
    __shared__ __align__(16) float4 tile[kWeightThreads / 32][2][kWideTokensWarp][32];
    const int b = blockIdx.z, h = blockIdx.y, n = clipped_length(a, b), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int t0 = (blockIdx.x * (kWeightThreads / 32) + warp) * kWideTokensWarp;
    dependents_wait();
    if (t0 >= n) return;
    const size_t bh = (size_t)b * a.c.heads + h;
    const float* x = a.logits + ((long long)bh * a.tokens + t0) * a.pitch;
    const float* row_lse = a.row_lse + bh * a.rows;
    const int steps = (a.rows + 127) / 128;
    auto fetch = [&](int i) {
        const int r = 128 * i + 4 * lane;
        if (i < steps && r < a.pitch) {             // (the pitch is a multiple of four here)
#pragma unroll
            for (int k = 0; k < kWideTokensWarp; ++k)
                if (t0 + k < n) cp_async_16(smem_u32(&tile[warp][i & 1][k][lane]), x + (long long)k * a.pitch + r);
        }
        cp_async_commit();
    };
    float sum[kWideTokensWarp];
#pragma unroll
    for (int k = 0; k < kWideTokensWarp; ++k) sum[k] = 0.f;
    fetch(0);
    for (int i = 0; i < steps; ++i) {
        fetch(i + 1);
        const int r = 128 * i + 4 * lane;
        float e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = r + j < a.rows ? for_weights(row_lse[r + j]) : 0.f;
        cp_async_wait<1>();
        __syncwarp();
#pragma unroll
        for (int k = 0; k < kWideTokensWarp; ++k) {
            const float4 l = tile[warp][i & 1][k][lane];
            const float w0 = weight_of(l.x, e[0]), w1 = weight_of(l.y, e[1]), w2 = weight_of(l.z, e[2]), w3 = weight_of(l.w, e[3]);
            sum[k] += r < a.rows ? w0 : 0.f;        // columns behind the last row hold anything
            sum[k] += r + 1 < a.rows ? w1 : 0.f;
            sum[k] += r + 2 < a.rows ? w2 : 0.f;
            sum[k] += r + 3 < a.rows ? w3 : 0.f;
        }
        __syncwarp();
    }
    float mine = 0.f;
#pragma unroll
    for (int k = 0; k < kWideTokensWarp; ++k) {
#pragma unroll
        for (int o = 16; o; o >>= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
        if (lane == k) mine = sum[k];
    }
    const int t = t0 + lane;
    if (lane < kWideTokensWarp && t < n) a.weights[b * a.ws[0] + h * a.ws[1] + t] = (a.add_to ? a.add_to[b * a.as[0] + h * a.as[1] + t] : 0.f) + mine;
}

// ---------------------------------------------------------------------------------------------------- host
struct AttnShape {
    int nt;                         // column groups of the narrow kernel, 0: the wide kernel
    int cluster;                    // narrow kernel: CTAs of a head, 0: all CTAs share all heads evenly
    int tiles, splits, pitch;
    long long tokens;
    size_t part_o, part_lse, row_lse, logits, bytes;
};

// Whether the CTAs of the narrow kernel take a head each (or a cluster of 2 to 8 a head, which joins its parts out of its shared
// memories) or share all heads' units evenly, with a second kernel for the joining.  Costs in units that a warp takes one after
// the other: 1.35 us at one group of rows, 1.7 at more.  Measured, us, 8 cache heads of 4 query heads, graph / eager:
//                                evenly        cluster of
//   1 sequence of    1000    14.4 / 23.6    8:  8.6 / 13.7
//                    4133    10.5 / 16.0    8: 11.9 / 14.6
//                    8192    11.7 / 15.7    8: 13.5 / 16.5
//                   16384    14.4 / 16.8    8: 19.6 / 21.7
//   16 sequences of  1000    19.7 / 22.6    1: 12.9 / 14.7
//                    8192    50.3 / 53.4    2: 44.8 / 47.4
//   1, weights       1000    15.0           8: 11.3
//                    4133    11.1           8: 14.8
// The rule goes by eager calls: at 4133 tokens it takes the cluster, which is the slower in a captured graph.  Lengths on the
// device may differ, so kRaggedUnits shuts out clusters whose warps would take more than eight units, even where the lengths
// turn out equal: 16 sequences of 8192 tokens take 50 us then instead of 45.
constexpr double kClusterJoin = 0.5;
constexpr double kSecondKernel = 3.25, kSecondAnyway = 0.4;     // its start, its launch on the host; with weights it runs all the same
constexpr double kCrossing = 2.5;                   // CTAs that work on two heads or sequences
constexpr int kRaggedUnits = 8;                     // where lengths may differ, the longest must not keep a cluster much longer than all the rest
static int cluster_of(long long pairs, long long units, int warps, bool weights, bool same) {
    const long long slots = 2 * kSMs, all = pairs * units, ctas = std::min(slots, (all + warps - 1) / warps);
    const double busy = warps == 8 ? 2.2 : 1.;      // a unit's time where HBM has all warps to serve
    const double load = busy * (double)all / (double)(slots * warps);
    const bool crossing = !same || pairs > ctas || ctas / pairs * pairs * 10 < ctas * 9;
    double best = (weights ? kSecondAnyway : kSecondKernel) + (crossing ? kCrossing : 0.) +
                  std::max((double)((all + slots * warps - 1) / (slots * warps)), load);
    int cluster = 0;
    for (int c = 1; c <= kMaxCluster && (c == 1 || pairs * c <= slots); c *= 2) {
        const long long turn = (units + c * warps - 1) / (c * warps), waves = (pairs * c + slots - 1) / slots;
        if (!same && turn > kRaggedUnits) continue;
        const double cost = std::max((double)(waves * turn), load) + (c > 1 ? kClusterJoin : 0.);
        if (cost < best) {
            best = cost;
            cluster = c;
        }
    }
    return cluster;
}

// `same`: sequences of one length
static AttnShape attention_shape(int batch, int hq, int heads, int n_q, int max_length, bool weights, bool same) {
    AttnShape s{};
    const long long rows = (long long)(hq / heads) * n_q, pairs = (long long)batch * heads;
    s.nt = rows <= kNarrowRows ? (int)((rows + 7) / 8) : 0;
    s.tiles = s.nt ? 1 : (int)((rows + kWideRows - 1) / kWideRows);
    long long parts;                // rows of partial results
    if (s.nt) {
        const int warps = narrow_warps(s.nt);
        const long long units = (long long)(max_length / kKv8Block) * (kKv8Block / kUnit) + warps;
        s.cluster = cluster_of(pairs, units, warps, weights, same);
        s.splits = s.cluster ? (int)(pairs * s.cluster) : (int)std::min<long long>(2 * kSMs, (pairs * units + warps - 1) / warps);
        parts = s.cluster ? 0 : (s.splits + pairs) * rows;
    } else {
        // one CTA an SM: the number of splits (of two tiles of tokens at least) that wastes least of its last wave; each
        // costs about as much again as two tiles (its start, its end and the joining)
        const long long ctas = pairs * s.tiles, tiles = (max_length + 127) / 128;
        double best = 1e30;
        for (long long k = 1; k <= std::max(1ll, tiles / 2) && k <= kSMs; ++k) {
            const double cost = (double)((ctas * k + kSMs - 1) / kSMs) * ((double)((tiles + k - 1) / k) + 2.0);
            if (cost < best - 1e-9) {
                best = cost;
                s.splits = (int)k;
            }
        }
        parts = s.splits > 1 ? pairs * rows * s.splits : 0;
    }
    s.pitch = rows <= 2 ? 2 : (int)((rows + 3) / 4 * 4);
    s.tokens = max_length;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    size_t at = 0;
    s.part_o = at;
    at = up(at + (size_t)parts * kKv8Dim * sizeof(float));
    s.part_lse = at;
    at = up(at + (size_t)(s.cluster && weights ? pairs * rows : parts) * sizeof(float));
    s.row_lse = at;
    if (weights && !s.nt) at = up(at + (size_t)pairs * rows * sizeof(float));
    s.logits = at;
    if (weights) at = up(at + (size_t)pairs * s.tokens * s.pitch * sizeof(float));
    s.bytes = at;
    return s;
}

static bool attention_sizes_ok(int batch, int hq, int heads, int n_q, int max_length) {
    return batch >= 1 && heads >= 1 && hq >= heads && hq % heads == 0 && n_q >= 1 && max_length >= 0 && (long long)hq * n_q <= (1 << 24);
}

template <int FMT, int NT, bool LOGITS>
static cudaError_t launch_narrow(const Kv8AttnArgs& a, cudaStream_t stream) {
    constexpr int bytes = narrow_warps(NT) * kRingSlots * kSlotBytes + (NT > 2 ? NT * 2048 + NT * 8 * sizeof(float) : 0);
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = allow_shared(kv8_attention_kernel<FMT, NT, LOGITS>, bytes, allowed);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = std::max(1, a.cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(a.splits);
    cfg.blockDim = dim3(narrow_warps(NT) * 32);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = a.cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kv8_attention_kernel<FMT, NT, LOGITS>, a);
}

template <int FMT, bool LOGITS>
static cudaError_t launch_narrow(const Kv8AttnArgs& a, int nt, cudaStream_t stream) {
    switch (nt) {
        case 1: return launch_narrow<FMT, 1, LOGITS>(a, stream);
        case 2: return launch_narrow<FMT, 2, LOGITS>(a, stream);
        default: return launch_narrow<FMT, 3, LOGITS>(a, stream);
    }
}

static cudaError_t launch_attention(const Kv8AttnArgs& a, const AttnShape& s, cudaStream_t stream) {
    if (!s.nt) return launch_attention_wide(a, s.tiles, stream);
    if (a.c.format == MINF_KV8_E4M3) return a.logits ? launch_narrow<MINF_KV8_E4M3, true>(a, s.nt, stream) : launch_narrow<MINF_KV8_E4M3, false>(a, s.nt, stream);
    return a.logits ? launch_narrow<MINF_KV8_INT8, true>(a, s.nt, stream) : launch_narrow<MINF_KV8_INT8, false>(a, s.nt, stream);
}

}  // namespace minf

using namespace minf;

extern "C" size_t minf_kv8_attention_scratch_bytes(int batch, int hq, int heads, int n_q, int max_length, int with_weights) {
    if (!attention_sizes_ok(batch, hq, heads, n_q, max_length)) return 0;
    // one sequence has one length; of several the caller may say so or not
    const size_t bytes = attention_shape(batch, hq, heads, n_q, max_length, with_weights != 0, true).bytes;
    return batch == 1 ? bytes : std::max(bytes, attention_shape(batch, hq, heads, n_q, max_length, with_weights != 0, false).bytes);
}

extern "C" int minf_kv8_attention(
    const minf_kv8_cache* cache, const void* q, const int64_t q_strides[3], void* o, const int64_t o_strides[3],
    int hq, int n_q, const int32_t* lengths, int length_all, int max_length, float sm_scale, float* lse,
    float* weights, const int64_t w_strides[2], const float* add_to, const int64_t add_strides[2],
    void* scratch, void* stream) {
    if (int rc = kv8_check(cache)) return rc;
    if (!q || !o || !q_strides || !o_strides || (weights && !w_strides) || (add_to && !add_strides)) return fail(MINF_E_ARG, "null pointer argument");
    if (!attention_sizes_ok(cache->batch, hq, cache->heads, n_q, max_length))
        return fail(MINF_E_ARG, "bad sizes (%d query heads over %d, %d queries, max_length %d)", hq, cache->heads, n_q, max_length);
    if (max_length > cache->capacity) return fail(MINF_E_ARG, "max_length %d is outside the cache of %d tokens", max_length, cache->capacity);
    if (!lengths && (length_all < 0 || length_all > max_length)) return fail(MINF_E_ARG, "length %d is outside [0, max_length %d]", length_all, max_length);
    if (add_to && !weights) return fail(MINF_E_ARG, "add_to without weights");
    const AttnShape s = attention_shape(cache->batch, hq, cache->heads, n_q, max_length, weights != nullptr, !lengths || cache->batch == 1);
    const long long a_rows = (long long)(hq / cache->heads) * n_q;
    if (s.bytes && !scratch) return fail(MINF_E_ARG, "scratch is needed (%zu bytes)", s.bytes);
    if (reinterpret_cast<uintptr_t>(scratch) & 15) return fail(MINF_E_ARG, "scratch must be 16-byte aligned");
    if (s.bytes > (size_t)1 << 46 || ((long long)max_length / kFinishTokens + 1 + a_rows) * cache->heads * cache->batch > 0x7fffffffll)
        return fail(MINF_E_UNSUPPORTED, "too large a call (%d sequences, %d heads, %lld rows)", cache->batch, cache->heads, a_rows);
    if ((long long)cache->heads * s.tiles > 65535) return fail(MINF_E_UNSUPPORTED, "too many query rows (%d heads of %d tiles)", cache->heads, s.tiles);
    Kv8AttnArgs a{};
    a.c = *cache;
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.o = static_cast<__nv_bfloat16*>(o);
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = q_strides[i];
        a.os[i] = o_strides[i];
        if (o_strides[i] % 4) return fail(MINF_E_ARG, "output strides must be multiples of 4 elements");
        if (q_strides[i] % 8) return fail(MINF_E_ARG, "query strides must be multiples of 8 elements");
    }
    if (reinterpret_cast<uintptr_t>(q) & 15) return fail(MINF_E_ARG, "the queries must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(o) & 7) return fail(MINF_E_ARG, "the output must be 8-byte aligned");
    a.group = hq / cache->heads;
    a.n_q = n_q;
    a.rows = a.group * n_q;
    a.lengths = lengths;
    a.length_all = length_all;
    a.max_length = max_length;
    a.scale_log2 = sm_scale * 1.4426950408889634f;
    a.splits = s.splits;
    a.cluster = s.cluster;
    char* base = static_cast<char*>(scratch);
    a.part_o = reinterpret_cast<float*>(base + s.part_o);
    a.part_lse = reinterpret_cast<float*>(base + s.part_lse);
    a.lse = lse;
    a.pitch = s.pitch;
    a.tokens = s.tokens;
    if (weights) {
        if (!s.nt) a.row_lse = reinterpret_cast<float*>(base + s.row_lse);
        a.logits = reinterpret_cast<float*>(base + s.logits);
        a.weights = weights;
        a.ws[0] = w_strides[0];
        a.ws[1] = w_strides[1];
        a.add_to = add_to;
        if (add_to) {
            a.as[0] = add_strides[0];
            a.as[1] = add_strides[1];
        }
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    cudaError_t e = launch_attention(a, s, st);
    if (e != cudaSuccess) return fail(MINF_E_CUDA, "launch of kv8_attention_kernel failed: %s", cudaGetErrorString(e));
    const long long pairs = (long long)cache->batch * cache->heads, rows = pairs * a.rows;
    a.chunk = kFinishTokens * (int)std::max(1ll, std::min(16ll, pairs * (max_length / kFinishTokens) / kFinishCtas));
    const long long chunks = weights ? ((long long)max_length + a.chunk - 1) / a.chunk : 0;
    if (s.cluster && !chunks) return MINF_OK;
    if (s.nt) {
        const dim3 grid((unsigned)(rows + pairs * chunks));
        e = narrow_warps(s.nt) == 8 ? launch_behind(kv8_finish_kernel<8>, grid, kFinishThreads, 0, st, a)
                                    : launch_behind(kv8_finish_kernel<4>, grid, kFinishThreads, 0, st, a);
        if (e != cudaSuccess) return fail(MINF_E_CUDA, "launch of kv8_finish_kernel failed: %s", cudaGetErrorString(e));
        return MINF_OK;
    }
    if (s.splits > 1) {
        e = launch_behind(kv8_finish_kernel<0>, dim3((unsigned)((rows + 7) / 8)), kFinishThreads, 0, st, a);
        if (e != cudaSuccess) return fail(MINF_E_CUDA, "launch of kv8_finish_kernel failed: %s", cudaGetErrorString(e));
    }
    if (chunks) {
        e = launch_behind(kv8_weights_kernel, dim3((unsigned)((max_length + kWideTokens - 1) / kWideTokens), cache->heads, cache->batch), kWeightThreads, 0, st, a);
        if (e != cudaSuccess) return fail(MINF_E_CUDA, "launch of kv8_weights_kernel failed: %s", cudaGetErrorString(e));
    }
    return MINF_OK;
}
