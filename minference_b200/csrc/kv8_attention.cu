// Attention over an 8-bit key/value cache (layout: kv8.cuh): decoding steps of one or a few tokens, and longer ones.
//
// For a row (query head, query token) with logits l_t = sm_scale log2(e) s_K,t (q . c_K,t) over the tokens it sees,
//   out = sum_t 2^(l_t - lse) s_V,t c_V,t,    lse = log2 sum_t 2^l_t
// in one pass over the cache.  The running maximum M is that of l_t + log2 s_V,t, so the numerators
// P_t = 2^(l_t + log2 s_V,t - M) are at most 1 and multiply the codes as they are, whatever the scales; the
// denominator is the sum over blocks of (sum P_t) / s_V.
//
// The products run on the tensor cores with the tokens as rows: S^T = K Q^T and O^T = V^T P^T, m16n8k16 in f16 with
// fp32 accumulation.  Eight query rows (a group of query heads that share a cache head, times the new tokens) fill the
// narrow side without padding to sixteen, and a code becomes an f16 value exactly.  Q is scaled by a power of two per
// row so that its bf16 values are f16 values (what is lost lies 2^-24 below the row's largest).  P is rounded to f16:
// half a step of 2^-11 relative, below the bf16 rounding of the output; sums and outputs are accumulated in fp32.
// The tail (bf16) takes bf16 products, with P as a sum of two bf16 numbers.
//
// The tokens of a sequence are split over CTAs and, inside one, over warps by blocks of 64; the parts are joined by
// their log-sum-exps in a second kernel.
#include "kv8_attention.cuh"

#include <math_constants.h>

#include <algorithm>

#include "sm100_ptx.cuh"

namespace minf {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kSlotBytes = kKv8Block * kKv8Dim;     // keys or values of a block
constexpr int kRingSlots = 3;
constexpr int kNarrowRows = 32;                     // rows per cache head this kernel takes
constexpr int kRingBytes = kAttnWarps * kRingSlots * kSlotBytes;

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
    const float lv = log2f(v_scale), inv_v = 1.f / v_scale;
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
            const int lim0 = all_see + r % a.n_q, lim1 = all_see + (r + 1) % a.n_q;
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
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
        }
        // the reference is raised on a jump of more than 2^8: P stays far below f16's largest, and outputs are rarely rescaled
        mx0 += lv;
        mx1 += lv;
        const bool up0 = mx0 > R.m[nt][0] + 8.f, up1 = mx1 > R.m[nt][1] + 8.f;
        if (__any_sync(0xffffffffu, up0 || up1)) {
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
        const float d0 = lv - (R.m[nt][0] == -CUDART_INF_F ? 0.f : R.m[nt][0]), d1 = lv - (R.m[nt][1] == -CUDART_INF_F ? 0.f : R.m[nt][1]);
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

template <int FMT, int NT, bool LOGITS>
__global__ void __launch_bounds__(kAttnThreads) kv8_attention_kernel(const __grid_constant__ Kv8AttnArgs a) {
    constexpr int SUB = 4 / NT;                     // sub-tiles of 16 tokens per softmax step: up to 16 logits a lane
    constexpr int PARTS = 4 / SUB;                  // softmax steps of a block
    constexpr bool kQShared = NT > 2;               // Q's fragments in shared memory (from there each is read once per sub-tile)
    extern __shared__ __align__(128) unsigned char ring_all[];
    const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, c = lane & 3;
    const int n = kv8_length(a.lengths, a.length_all, b, a.max_length, a.c.status);
    const size_t bh = (size_t)b * a.c.heads + h;
    const int full = n / kKv8Block;                 // complete blocks
    // the last split takes the tail too, which keeps all four warps busy: it counts as four blocks
    const int units = full + (n % kKv8Block ? kAttnWarps : 0);
    const int blk_lo = min(full, (int)((long long)units * split / a.splits)), blk_hi = min(full, (int)((long long)units * (split + 1) / a.splits));
    const int all_see = n - a.n_q + 1;              // tokens below this are seen by every row

    // The warp's own ring of three slots of 8 KB: keys of a block, values of it, keys of its next block, ...; two
    // copies are in flight while the third is used.  16-byte chunk ch of row r lies at ch ^ (r & 7).
    unsigned char* const ring = ring_all + warp * (kRingSlots * kSlotBytes);
    const uint32_t ring_u = smem_u32(ring);
    const uint32_t put0 = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4), put1 = (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3) + 4)) << 4);
    auto fetch = [&](int slot, const uint8_t* src) {
        src += lane * 16;
        const uint32_t dst = ring_u + slot * kSlotBytes;
#pragma unroll
        for (int i = 0; i < 16; ++i) cp_async_16(dst + 512 * i + ((i & 1) ? put1 : put0), src + 512 * i);
    };
    const float* ks = a.c.k_scale + bh * (a.c.capacity / kKv8Block);
    const float* vs = a.c.v_scale + bh * (a.c.capacity / kKv8Block);
    const size_t first = (bh * (a.c.capacity / kKv8Block) + blk_lo + warp) * kSlotBytes;
    const uint8_t* next_k = static_cast<const uint8_t*>(a.c.k) + first;
    const uint8_t* next_v = static_cast<const uint8_t*>(a.c.v) + first;
    float k_scale = 1.f, v_scale = 1.f;
    if (blk_lo + warp < blk_hi) {
        fetch(0, next_k);
        cp_async_commit();
        fetch(1, next_v);
        k_scale = ks[blk_lo + warp];
        v_scale = vs[blk_lo + warp];
    } else {
        cp_async_commit();
    }
    cp_async_commit();

    // Q^T fragments: column g of group nt, dims of step s: 64 (s / 4) + 16 c + 4 (s % 4) + {0, 1 | 2, 3}
    Rows<NT> R;
    uint32_t qf[kQShared ? 1 : NT][8][2];
    uint2* const q_sm = reinterpret_cast<uint2*>(ring_all + kRingBytes);        // [nt][step][lane]
    float q_unit[NT];                               // power of two the row was divided by
    // eight dims of row 8 nt + g from dim d on (zeros behind the last row)
    auto q_load = [&](int nt, int d, float (&v)[8]) {
        const int r = 8 * nt + g;
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (r < a.rows) x = *reinterpret_cast<const uint4*>(a.q + b * a.qs[0] + (long long)(h * a.group + r / a.n_q) * a.qs[1] + (long long)(r % a.n_q) * a.qs[2] + d);
        bf16x8_to_values(x, v);
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float top = 0.f;
        float x[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q_load(nt, 64 * (i >> 1) + 16 * c + 8 * (i & 1), x[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float m = fabsf(x[i][e]);
                if (m < CUDART_INF_F) top = fmaxf(top, m);
            }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int e = 0;
        if (top > 0.f) frexpf(top, &e);             // top < 2^e: scaled to below 2^8, so that the smallest products count too
        e = max(min(e - 8, 100), -100);
        const float inv = exp2f((float)-e);
        q_unit[nt] = exp2f((float)e);
#pragma unroll
        for (int st = 0; st < 8; ++st) {
            const float* v = &x[st >> 1][4 * (st & 1)];
            const uint32_t b0 = pack_half2(v[0] * inv, v[1] * inv), b1 = pack_half2(v[2] * inv, v[3] * inv);
            if constexpr (kQShared) {
                if (warp == 0) q_sm[(nt * 8 + st) * 32 + lane] = make_uint2(b0, b1);
            } else {
                qf[nt][st][0] = b0;
                qf[nt][st][1] = b1;
            }
        }
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
            R.mul[nt][cc] = a.scale_log2 * __shfl_sync(0xffffffffu, q_unit[nt], 4 * (2 * c + cc));
            R.m[nt][cc] = -CUDART_INF_F;
            R.l[nt][cc] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) R.o[nt][i][k] = 0.f;
    }
    if (kQShared) __syncthreads();
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
    for (int blk = blk_lo + warp; blk < blk_hi; blk += kAttnWarps) {
        const bool more = blk + kAttnWarps < blk_hi;
        const bool masked = (blk + 1) * kKv8Block > all_see;
        const float ksc = k_scale, vsc = v_scale;
        next_k += kHop;
        next_v += kHop;
        const int slot_v = slot == 2 ? 0 : slot + 1, slot_n = slot_v == 2 ? 0 : slot_v + 1;
        if (more) {
            fetch(slot_n, next_k);
            k_scale = ks[blk + kAttnWarps];
            v_scale = vs[blk + kAttnWarps];
        }
        cp_async_commit();
        cp_async_wait<2>();
        __syncwarp();
        const unsigned char* kb = ring + slot * kSlotBytes;
        const unsigned char* vb = ring + slot_v * kSlotBytes;
        bool v_here = false;
#pragma unroll 1
        for (int part = 0; part < PARTS; ++part) {
            const int t0 = blk * kKv8Block + part * SUB * 16;
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
        // both slots are free: the values of the next block take the one the keys were in
        if (more) fetch(slot, next_v);
        cp_async_commit();
        slot = slot_n;
    }

    // the tail: the last split's warps take 16 of its tokens each
    const int t0 = full * kKv8Block + 16 * warp;
    if (split == a.splits - 1 && t0 < n) {
        const __nv_bfloat16* kt = static_cast<const __nv_bfloat16*>(a.c.k_tail) + (bh * kKv8Block + 16 * warp) * kKv8Dim;
        const __nv_bfloat16* vt = static_cast<const __nv_bfloat16*>(a.c.v_tail) + (bh * kKv8Block + 16 * warp) * kKv8Dim;
        float s[1][NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[0][nt][e] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {               // 16 dims of a lane quad: two steps
            const int d = 64 * (i >> 1) + 16 * c + 8 * (i & 1);
            const uint4 x = *reinterpret_cast<const uint4*>(kt + g * kKv8Dim + d), y = *reinterpret_cast<const uint4*>(kt + (g + 8) * kKv8Dim + d);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float v[8];
                q_load(nt, d, v);
                const float inv = 1.f / q_unit[nt];
                mma_bf16(s[0][nt], x.x, y.x, x.y, y.y, pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
                mma_bf16(s[0][nt], x.z, y.z, x.w, y.w, pack_bf16x2(v[4] * inv, v[5] * inv), pack_bf16x2(v[6] * inv, v[7] * inv));
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

    // Join the warps, eight rows at a time.  Where a row did not see all of a block's tokens, values that are infinite or
    // NaN were left out of the products (zero times them would not be zero) and are added here to the rows that see them.
    const bool any_bad = __syncthreads_or(bad);     // (and the rings are read out)
    float (*sm_o)[8][kKv8Dim] = reinterpret_cast<float (*)[8][kKv8Dim]>(ring_all);
    float (*sm_lse)[8] = reinterpret_cast<float (*)[8]>(ring_all + kAttnWarps * 8 * kKv8Dim * sizeof(float));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int cc = 0; cc < 2; ++cc) {
            float l = R.l[nt][cc];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            const float inv = l == 0.f ? 0.f : 1.f / l;
            if (g == 0) sm_lse[warp][2 * c + cc] = l == 0.f ? -CUDART_INF_F : (R.m[nt][cc] == -CUDART_INF_F ? l : R.m[nt][cc] + log2f(l));
            float* dst = &sm_o[warp][2 * c + cc][16 * g];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(dst + 4 * i) = make_float4(R.o[nt][2 * i][cc] * inv, R.o[nt][2 * i][2 + cc] * inv,
                                                                      R.o[nt][2 * i + 1][cc] * inv, R.o[nt][2 * i + 1][2 + cc] * inv);
        }
        __syncthreads();
#pragma unroll 1
        for (int i = threadIdx.x; i < 8 * 32; i += kAttnThreads) {
            const int rr = i >> 5, d = (i & 31) * 4, r = 8 * nt + rr;
            if (r >= a.rows) continue;
            float top = sm_lse[0][rr];
#pragma unroll
            for (int w = 1; w < kAttnWarps; ++w) top = fmaxf(top, sm_lse[w][rr]);
            float sum = 0.f;
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kAttnWarps; ++w) {
                const float e = sm_lse[w][rr];
                if (e == -CUDART_INF_F) continue;
                const float f = exp2f(e - top);
                const float4 x = *reinterpret_cast<const float4*>(&sm_o[w][rr][d]);
                sum += f;
                acc[0] = fmaf(f, x.x, acc[0]);
                acc[1] = fmaf(f, x.y, acc[1]);
                acc[2] = fmaf(f, x.z, acc[2]);
                acc[3] = fmaf(f, x.w, acc[3]);
            }
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] *= inv;
            if (any_bad) {
                const int lo = max(blk_lo, max(all_see, 0) / kKv8Block) * kKv8Block, lim = all_see + r % a.n_q;
                const int hi = min(split == a.splits - 1 ? n : blk_hi * kKv8Block, lim);
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
            const float lse = sum == 0.f ? -CUDART_INF_F : top + log2f(sum);
            const size_t row = bh * a.rows + r;
            if (a.splits > 1) {
                *reinterpret_cast<float4*>(a.part_o + (row * a.splits + split) * kKv8Dim + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                if (d == 0) a.part_lse[row * a.splits + split] = lse;
            } else {
                const int hq = h * a.group + r / a.n_q, t = r % a.n_q;
                __nv_bfloat16* o = a.o + b * a.os[0] + hq * a.os[1] + t * a.os[2] + d;
                *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
                if (d == 0) {
                    if (a.lse) a.lse[((size_t)b * a.c.heads * a.group + hq) * a.n_q + t] = lse;
                    if (a.row_lse) a.row_lse[row] = lse;
                }
            }
        }
        __syncthreads();
    }
}

// The splits of one row joined: four warps take every fourth split, a lane four dims.
__global__ void __launch_bounds__(128) kv8_combine_kernel(const __grid_constant__ Kv8AttnArgs a) {
    __shared__ float4 sm[4][32];
    __shared__ float sm_sum[4];
    const size_t row = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float* lse = a.part_lse + row * a.splits;
    float top = -CUDART_INF_F;
    for (int i = lane; i < a.splits; i += 32) top = fmaxf(top, lse[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = warp; i < a.splits; i += 4) {
        const float e = lse[i];
        if (e == -CUDART_INF_F) continue;
        const float f = exp2f(e - top);
        const float4 x = *reinterpret_cast<const float4*>(a.part_o + (row * a.splits + i) * kKv8Dim + 4 * lane);
        sum += f;
        acc.x = fmaf(f, x.x, acc.x);
        acc.y = fmaf(f, x.y, acc.y);
        acc.z = fmaf(f, x.z, acc.z);
        acc.w = fmaf(f, x.w, acc.w);
    }
    sm[warp][lane] = acc;
    if (lane == 0) sm_sum[warp] = sum;
    __syncthreads();
    if (warp) return;
    sum = sm_sum[0] + sm_sum[1] + sm_sum[2] + sm_sum[3];
    acc = sm[0][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
        const float4 x = sm[w][lane];
        acc.x += x.x;
        acc.y += x.y;
        acc.z += x.z;
        acc.w += x.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const size_t bh = row / a.rows;
    const int r = (int)(row % a.rows), b = (int)(bh / a.c.heads), h = (int)(bh % a.c.heads);
    const int hq = h * a.group + r / a.n_q, t = r % a.n_q;
    __nv_bfloat16* o = a.o + b * a.os[0] + hq * a.os[1] + t * a.os[2] + 4 * lane;
    *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
    if (lane == 0) {
        const float e = sum == 0.f ? -CUDART_INF_F : top + log2f(sum);
        if (a.lse) a.lse[((size_t)b * a.c.heads * a.group + hq) * a.n_q + t] = e;
        if (a.row_lse) a.row_lse[row] = e;
    }
}

// Attention weight of every token of a head: the probabilities of the head's rows, summed in their order.
__global__ void __launch_bounds__(256) kv8_weights_kernel(const __grid_constant__ Kv8AttnArgs a) {
    const int b = blockIdx.z, h = blockIdx.y;
    const int n = kv8_length(a.lengths, a.length_all, b, a.max_length, a.c.status);
    const int t = blockIdx.x * 256 + threadIdx.x;
    if (t >= n) return;
    const size_t bh = (size_t)b * a.c.heads + h;
    const float* x = a.logits + ((long long)bh * a.tokens + t) * a.pitch;
    const float* e = a.row_lse + bh * a.rows;
    float sum = 0.f;
    for (int r = 0; r < a.rows; r += 2) {
        const float2 l = *reinterpret_cast<const float2*>(x + r);
        const float e0 = e[r];
        sum += l.x == -CUDART_INF_F ? 0.f : exp2f(l.x - e0);
        if (r + 1 < a.rows) sum += l.y == -CUDART_INF_F ? 0.f : exp2f(l.y - e[r + 1]);
    }
    const float was = a.add_to ? a.add_to[b * a.as[0] + h * a.as[1] + t] : 0.f;
    a.weights[b * a.ws[0] + h * a.ws[1] + t] = was + sum;
}

// ---------------------------------------------------------------------------------------------------- host
struct AttnShape {
    int nt, tiles, splits, pitch;
    long long tokens;
    size_t part_o, part_lse, row_lse, logits, bytes;
};

static AttnShape attention_shape(int batch, int hq, int heads, int n_q, int max_length, bool weights) {
    AttnShape s{};
    const long long rows = (long long)(hq / heads) * n_q;
    s.nt = rows <= kNarrowRows ? (int)((rows + 7) / 8) : 0;
    s.tiles = s.nt ? 1 : (int)((rows + kWideRows - 1) / kWideRows);
    const long long ctas = (long long)batch * heads * s.tiles;
    const long long blocks = max_length / kKv8Block;
    if (s.nt) {
        long long splits = (2 * kSMs + ctas - 1) / ctas;
        splits = std::min(splits, (blocks + kAttnWarps - 1) / kAttnWarps);
        s.splits = (int)std::max(splits, 1ll);
    } else {
        // one CTA an SM: the number of splits (of two tiles of tokens at least) that wastes least of its last wave; each
        // costs about as much again as two tiles (its start, its end and the joining)
        const long long tiles = (max_length + 127) / 128;
        double best = 1e30;
        for (long long k = 1; k <= std::max(1ll, tiles / 2) && k <= kSMs; ++k) {
            const double cost = (double)((ctas * k + kSMs - 1) / kSMs) * ((double)((tiles + k - 1) / k) + 2.0);
            if (cost < best - 1e-9) {
                best = cost;
                s.splits = (int)k;
            }
        }
    }
    s.pitch = (int)((rows + 1) / 2 * 2);
    s.tokens = max_length;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    const size_t all = (size_t)batch * heads * rows;
    size_t at = 0;
    s.part_o = at;
    if (s.splits > 1) at = up(at + all * s.splits * kKv8Dim * sizeof(float));
    s.part_lse = at;
    if (s.splits > 1) at = up(at + all * s.splits * sizeof(float));
    s.row_lse = at;
    if (weights) at = up(at + all * sizeof(float));
    s.logits = at;
    if (weights) at = up(at + (size_t)batch * heads * s.tokens * s.pitch * sizeof(float));
    s.bytes = at;
    return s;
}

static bool attention_sizes_ok(int batch, int hq, int heads, int n_q, int max_length) {
    return batch >= 1 && heads >= 1 && hq >= heads && hq % heads == 0 && n_q >= 1 && max_length >= 0 && (long long)hq * n_q <= (1 << 24);
}

template <int FMT, int NT, bool LOGITS>
static cudaError_t launch_narrow(const Kv8AttnArgs& a, cudaStream_t stream) {
    constexpr int bytes = kRingBytes + (NT > 2 ? NT * 2048 : 0);
    // per device, and cheap: every call sets it
    const cudaError_t e = cudaFuncSetAttribute(kv8_attention_kernel<FMT, NT, LOGITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    kv8_attention_kernel<FMT, NT, LOGITS><<<dim3(a.splits, a.c.heads, a.c.batch), kAttnThreads, bytes, stream>>>(a);
    return cudaGetLastError();
}

template <int FMT, bool LOGITS>
static cudaError_t launch_narrow(const Kv8AttnArgs& a, int nt, cudaStream_t stream) {
    switch (nt) {
        case 1: return launch_narrow<FMT, 1, LOGITS>(a, stream);
        case 2: return launch_narrow<FMT, 2, LOGITS>(a, stream);
        case 3: return launch_narrow<FMT, 3, LOGITS>(a, stream);
        default: return launch_narrow<FMT, 4, LOGITS>(a, stream);
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
    return attention_shape(batch, hq, heads, n_q, max_length, with_weights != 0).bytes;
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
    const AttnShape s = attention_shape(cache->batch, hq, cache->heads, n_q, max_length, weights != nullptr);
    if (s.bytes && !scratch) return fail(MINF_E_ARG, "scratch is needed (%zu bytes)", s.bytes);
    if (reinterpret_cast<uintptr_t>(scratch) & 15) return fail(MINF_E_ARG, "scratch must be 16-byte aligned");
    if ((long long)cache->heads * s.tiles > 65535) return fail(MINF_E_UNSUPPORTED, "too many query rows (%d heads of %d tiles)", cache->heads, s.tiles);
    Kv8AttnArgs a{};
    a.c = *cache;
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.o = static_cast<__nv_bfloat16*>(o);
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = q_strides[i];
        a.os[i] = o_strides[i];
        if (o_strides[i] % 4) return fail(MINF_E_ARG, "output strides must be multiples of 4 elements");
    }
    if (reinterpret_cast<uintptr_t>(o) & 7) return fail(MINF_E_ARG, "the output must be 8-byte aligned");
    a.group = hq / cache->heads;
    a.n_q = n_q;
    a.rows = a.group * n_q;
    a.lengths = lengths;
    a.length_all = length_all;
    a.max_length = max_length;
    a.scale_log2 = sm_scale * 1.4426950408889634f;
    a.splits = s.splits;
    char* base = static_cast<char*>(scratch);
    a.part_o = reinterpret_cast<float*>(base + s.part_o);
    a.part_lse = reinterpret_cast<float*>(base + s.part_lse);
    a.lse = lse;
    a.pitch = s.pitch;
    a.tokens = s.tokens;
    if (weights) {
        a.row_lse = reinterpret_cast<float*>(base + s.row_lse);
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
    const cudaError_t e = launch_attention(a, s, st);
    if (e != cudaSuccess) return fail(MINF_E_CUDA, "launch of kv8_attention_kernel failed: %s", cudaGetErrorString(e));
    if (s.splits > 1) {
        kv8_combine_kernel<<<(unsigned)((size_t)cache->batch * cache->heads * a.rows), 128, 0, st>>>(a);
        MINF_LAUNCH_OK("kv8_combine_kernel");
    }
    if (weights && max_length > 0) {
        kv8_weights_kernel<<<dim3((max_length + 255) / 256, cache->heads, cache->batch), 256, 0, st>>>(a);
        MINF_LAUNCH_OK("kv8_weights_kernel");
    }
    return MINF_OK;
}
