// Attention over an 8-bit cache for many query rows per cache head (several new tokens, large groups): the formulas and
// the splitting of kv8_attention.cu, on the tcgen05 tensor cores.
//
// One CTA owns 128 rows of a head and a stretch of its tokens, in tiles of 128.  Warp roles:
//   warps 0-3, 4-7   softmax of the even / odd tiles, a thread per row.  Each group keeps its own maximum, sum and
//                    output (S and O in TMEM, P written over S as f16), so the softmax of one tile runs under the
//                    products of the other; the two results are joined at the end.
//   warps 8-11       turn codes into f16 operands: cp.async into a ring of four 16 KB tiles, three of them in flight,
//                    then conversion into the 128-byte-swizzled K and V stages.  A thread converts what it copied
//                    itself, so the ring needs no barrier.
//   warp 12          issues the MMAs.
// (Four warps at most share a scheduler, so a thread may hold 128 registers.)
// TMEM: O and S of the two groups, 4 x 128 columns.
//
// The tail's bf16 values become f16 by a power of two for the block (what is lost lies 2^-33 below its largest value).
// In tiles that some row does not see to its end, values that are infinite or NaN are left out of the product (zero
// times them would reach rows that do not see them) and added to the rows that do at the end.
//
// Bound: with 128 live rows the tensor pipe, 16 products of 64 cycles a tile; with few rows the 32 KB a tile takes from
// HBM (about 1400 cycles of an SM's share), under which 1024 cycles of padded products hide.
#include "kv8_attention.cuh"

#include <math_constants.h>

#include "sm100_ptx.cuh"

namespace minf {

constexpr int kWideTile = 128;                      // tokens of a tile
constexpr uint32_t kOperand = 128 * 256;            // 128 rows x 128 f16
constexpr uint32_t kRawTile = 128 * 128;            // codes of a tile
constexpr int kRawSlots = 4;
constexpr uint32_t kWQOff = 0, kWKOff = kOperand, kWVOff = 3 * kOperand, kWRawOff = 5 * kOperand;
constexpr uint32_t kWCtlOff = kWRawOff + kRawSlots * kRawTile;
constexpr int kConvWarps = 4, kMmaWarp = 8 + kConvWarps;
constexpr int kWideThreads = (kMmaWarp + 1) * 32;
constexpr int kConvThreads = kConvWarps * 32;
constexpr int kConvParts = kRawTile / (16 * kConvThreads);     // 16-byte pieces of a tile a thread converts

struct WideCtl {
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], tail_ready, o_done;
    uint32_t tmem_base;
    int abort;
    int bad;                        // a value left out of the product because it is not finite
    float tail_scale[2];            // of the tail's keys and values
    float red[2][kConvWarps];
    float unit[kWideRows];          // power of two a query row was divided by
    float lse[kWideRows];
};
static_assert(kWCtlOff + sizeof(WideCtl) <= 232448, "shared memory of one CTA");

__device__ __forceinline__ uint32_t pack_half2_rn(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void st_shared_16(uint32_t dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_16(uint32_t src) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
    return v;
}
// byte offset of 16-byte chunk ch (8 f16, 0..15) of row r in an operand stage
__device__ __forceinline__ uint32_t operand_at(int r, int ch) {
    return (uint32_t)(ch >> 3) * 16384u + (uint32_t)r * 128u + (uint32_t)(((ch ^ r) & 7) << 4);
}
// Halves that are infinite or NaN become zero; true if there were any.
__device__ __forceinline__ bool drop_not_finite(uint32_t& x) {
    const bool lo = (x & 0x7c00u) == 0x7c00u, hi = (x & 0x7c000000u) == 0x7c000000u;
    if (lo) x &= 0xffff0000u;
    if (hi) x &= 0x0000ffffu;
    return lo || hi;
}

// Maximum of l + log2 s_V over a tile's 128 tokens for the thread's row: S in 128 columns at t_s, logit = S * f of the
// token's half (f >= 0: the sign of the softmax scale is in Q).  MASKED: only the tokens below `lim` of the tile; the
// logits of those below `end` are written out where LOGITS asks for them.
template <bool MASKED, bool LOGITS>
__device__ __forceinline__ float row_max(uint32_t t_s, const float (&f)[2], const float (&lv)[2], int lim, int end, float* logits, int pitch) {
    float mx = -CUDART_INF_F;
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
        const float fh = half ? f[1] : f[0], lh = half ? lv[1] : lv[0];
        float m4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
        uint32_t s[2][32];
        tmem_ld32(t_s + 64 * half, s[0]);
        tmem_ld32(t_s + 64 * half + 32, s[1]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
                if constexpr (MASKED) {
                    const int t = 64 * half + 32 * c + k;
                    if (t >= lim) s[c][k] = 0xff800000u;                        // -inf
                    if (t + 1 >= lim) s[c][k + 1] = 0xff800000u;
                    if constexpr (LOGITS) {
                        if (logits && t < end) logits[(long long)t * pitch] = t >= lim ? -CUDART_INF_F : __uint_as_float(s[c][k]) * fh;
                        if (logits && t + 1 < end) logits[(long long)(t + 1) * pitch] = t + 1 >= lim ? -CUDART_INF_F : __uint_as_float(s[c][k + 1]) * fh;
                    }
                }
                m4[(k >> 1) & 3] = max3(m4[(k >> 1) & 3], __uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1]));
            }
        const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        if (m != -CUDART_INF_F) mx = fmaxf(mx, fmaf(m, fh, lh));                // (-inf times a scale of zero would be NaN)
    }
    return mx;
}

// P = 2^(l + log2 s_V - ref) of the row, as f16 over the first half of S's columns; the denominator's part is added to l_sum.
template <bool MASKED>
__device__ __forceinline__ void row_numerators(uint32_t t_s, const float (&f)[2], const float (&lv)[2], const float (&inv_v)[2], float ref, int lim, float& l_sum) {
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
        const float fh = half ? f[1] : f[0], d = (half ? lv[1] : lv[0]) - ref;
        const uint64_t f2 = pack_f32x2(fh, fh), d2 = pack_f32x2(d, d);
        uint64_t sum2[2] = {0ull, 0ull};
        uint32_t s[2][32];
        tmem_ld32(t_s + 64 * half, s[0]);
        tmem_ld32(t_s + 64 * half + 32, s[1]);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t p[16];
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
                float x0, x1;
                unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[c][k]), __uint_as_float(s[c][k + 1])), f2, d2), x0, x1);
                if constexpr (MASKED) {
                    const int t = 64 * half + 32 * c + k;
                    if (t >= lim) x0 = -CUDART_INF_F;
                    if (t + 1 >= lim) x1 = -CUDART_INF_F;
                }
                x0 = fast_exp2(x0);
                x1 = fast_exp2(x1);
                sum2[(k >> 1) & 1] = add_f32x2(sum2[(k >> 1) & 1], pack_f32x2(x0, x1));
                p[k >> 1] = pack_half2_rn(x0, x1);
            }
            tmem_st16(t_s + 32 * half + 16 * c, p);                             // over columns the thread has read
        }
        float a0, a1;
        unpack_f32x2(add_f32x2(sum2[0], sum2[1]), a0, a1);
        l_sum = fmaf(a0 + a1, half ? inv_v[1] : inv_v[0], l_sum);
    }
}

template <int FMT, bool LOGITS>
__global__ void __launch_bounds__(kWideThreads, 1) kv8_attention_wide_kernel(const __grid_constant__ Kv8AttnArgs a, const int tiles) {
    extern __shared__ __align__(1024) unsigned char smem[];
    WideCtl* ctl = reinterpret_cast<WideCtl*>(smem + kWCtlOff);
    const uint32_t smem_base = smem_u32(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x, b = blockIdx.z, h = blockIdx.y / tiles, row0 = (blockIdx.y % tiles) * kWideRows;
    const int n = kv8_length(a.lengths, a.length_all, b, a.max_length, a.c.status);
    const size_t bh = (size_t)b * a.c.heads + h;
    const int full = n / kKv8Block;
    const int all_see = n - a.n_q + 1;
    // tokens that no row of this CTA sees are left out, unless the weights want their logits
    const int last_row = min(row0 + kWideRows, a.rows) - 1;
    const int last_token = last_row / a.n_q > row0 / a.n_q ? a.n_q - 1 : last_row % a.n_q;
    const int end = LOGITS ? n : max(min(n, all_see + last_token), 0);
    const int total = (end + kWideTile - 1) / kWideTile;
    const int j_lo = (int)((long long)total * split / a.splits), j_hi = (int)((long long)total * (split + 1) / a.splits);
    const int count = j_hi - j_lo;                  // this CTA's tiles
    const bool has_tail = j_hi == (n + kWideTile - 1) / kWideTile && n % kKv8Block && count > 0;

    dependents_launch();
    auto bar = [&](const unsigned long long* p) { return smem_u32(p); };
    volatile int* abort_flag = &ctl->abort;
    if (threadIdx.x == 0) {
        for (int s = 0; s < 2; ++s) {
            mbar_init(bar(&ctl->k_full[s]), kConvWarps);
            mbar_init(bar(&ctl->v_full[s]), kConvWarps);
            mbar_init(bar(&ctl->k_empty[s]), 1);
            mbar_init(bar(&ctl->v_empty[s]), 1);
            mbar_init(bar(&ctl->s_full[s]), 1);
            mbar_init(bar(&ctl->p_full[s]), 128);   // the rows' threads
        }
        mbar_init(bar(&ctl->tail_ready), kConvWarps);
        mbar_init(bar(&ctl->o_done), 1);
        ctl->abort = 0;
        ctl->bad = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&ctl->tmem_base), 512);
        tmem_relinquish();
    }
    if (warp < 4) {                                 // the query rows, a thread each
        const int r = row0 + threadIdx.x;
        uint4 x[16];
        float top = 0.f;
        if (r < a.rows) {
            const uint4* q = reinterpret_cast<const uint4*>(a.q + b * a.qs[0] + (long long)(h * a.group + r / a.n_q) * a.qs[1] + (long long)(r % a.n_q) * a.qs[2]);
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = q[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v[8];
            bf16x8_to_values(x[i], v);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float m = fabsf(v[k]);
                if (m < CUDART_INF_F) top = fmaxf(top, m);
            }
        }
        int e = 0;
        if (top > 0.f) frexpf(top, &e);
        e = max(min(e - 8, 100), -100);
        const float inv = a.scale_log2 < 0.f ? -exp2f((float)-e) : exp2f((float)-e);
        ctl->unit[threadIdx.x] = exp2f((float)e);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float v[8];
            bf16x8_to_values(x[i], v);
            st_shared_16(smem_base + kWQOff + operand_at(threadIdx.x, i), pack_half2_rn(v[0] * inv, v[1] * inv), pack_half2_rn(v[2] * inv, v[3] * inv),
                         pack_half2_rn(v[4] * inv, v[5] * inv), pack_half2_rn(v[6] * inv, v[7] * inv));
        }
        fence_proxy_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;

    float m_ref = -CUDART_INF_F, l_sum = 0.f;       // of a softmax thread's row
    bool ok = true;
    if (warp == kMmaWarp) {
        // ------------------------------------------------------------------------------------------ products
        auto wait = [&](const unsigned long long* p, int parity) { return __all_sync(0xffffffffu, mbar_wait(bar(p), parity, abort_flag)) != 0; };
        constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
        auto desc = [](uint32_t lo) { return (static_cast<uint64_t>(kDescHi) << 32) | lo; };
        auto issue_s = [&](int i) {
            ok = ok && wait(&ctl->k_full[i & 1], (i >> 1) & 1);
            if (!ok) return;
            constexpr uint32_t idesc = umma_idesc(128, 128, false, false, false);
            const uint32_t d = tmem + (i & 1) * 256 + 128;
            const uint32_t q_lo = ((smem_base + kWQOff) >> 4) | (1u << 16), k_lo = ((smem_base + kWKOff + (i & 1) * kOperand) >> 4) | (1u << 16);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < 8; ++kk) {
                    const uint32_t adv = (kk >> 2) * (16384 >> 4) + (kk & 3) * (32 >> 4);
                    umma_ss(d, desc(q_lo + adv), desc(k_lo + adv), idesc, kk > 0);
                }
                umma_commit(bar(&ctl->s_full[i & 1]));
                umma_commit(bar(&ctl->k_empty[i & 1]));
            }
        };
        auto issue_pv = [&](int i) {
            ok = ok && wait(&ctl->v_full[i & 1], (i >> 1) & 1);
            ok = ok && wait(&ctl->p_full[i & 1], (i >> 1) & 1);
            if (!ok) return;
            tc_fence_after();
            constexpr uint32_t idesc = umma_idesc(128, 128, false, false, true);
            const uint32_t d = tmem + (i & 1) * 256, p = d + 128;
            const uint32_t v_lo = ((smem_base + kWVOff + (i & 1) * kOperand) >> 4) | ((16384u >> 4) << 16);
            if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < 8; ++kk) umma_ts(d, p + kk * 8, desc(v_lo + kk * (2048 >> 4)), idesc, (i > 1 || kk > 0) ? 1u : 0u);
                umma_commit(bar(&ctl->v_empty[i & 1]));
            }
        };
        if (count > 0) issue_s(0);
        if (count > 1) issue_s(1);
        for (int i = 0; i < count && ok; ++i) {
            issue_pv(i);
            if (i + 2 < count) issue_s(i + 2);
        }
        if (ok && elect_one()) {
            if (count > 0) umma_commit(bar(&ctl->o_done));
            else mbar_arrive(bar(&ctl->o_done));
        }
    } else if (warp >= 8) {
        // ---------------------------------------------------------------------------------------- conversion
        const int dw = warp - 8, tid = threadIdx.x - 256;
        const uint8_t* codes[2] = {static_cast<const uint8_t*>(a.c.k) + bh * a.c.capacity * kKv8Dim, static_cast<const uint8_t*>(a.c.v) + bh * a.c.capacity * kKv8Dim};
        const __nv_bfloat16* tails[2] = {static_cast<const __nv_bfloat16*>(a.c.k_tail) + bh * kKv8Block * kKv8Dim,
                                         static_cast<const __nv_bfloat16*>(a.c.v_tail) + bh * kKv8Block * kKv8Dim};
        constexpr int kRowHop = kConvThreads / 8, kPartBytes = kConvThreads * 16;
        const int row = tid >> 3, ch = tid & 7;                         // rows row + kRowHop u, 16 codes from 16 ch
        const uint32_t raw = smem_base + kWRawOff + tid * 16;
        // items in the order the products want them: K0 K1 V0 K2 V1 ... ; number m = 2 i (values) or 2 i - 1 (keys)
        auto which_of = [](int m) { return m == 0 || (m & 1) ? 0 : 1; };
        auto tile_of = [](int m) { return m == 0 ? 0 : (m & 1) ? (m + 1) / 2 : m / 2 - 1; };
        const int items = 2 * count + 1;
        auto fetch = [&](int m) {
            const int i = tile_of(m);
            if (m < items && i < count) {
                const int t0 = (j_lo + i) * kWideTile;
                const uint8_t* src = codes[which_of(m)] + (size_t)t0 * kKv8Dim + tid * 16;
                const uint32_t dst = raw + (m & (kRawSlots - 1)) * kRawTile;
#pragma unroll
                for (int u = 0; u < kConvParts; ++u)
                    if (t0 + row + kRowHop * u < full * kKv8Block) cp_async_16(dst + u * kPartBytes, src + u * kPartBytes);
            }
            cp_async_commit();
        };
        for (int m = 0; m < kRawSlots - 1; ++m) fetch(m);
        if (has_tail) {                             // the tail's scales, before its tile is due
            float top[2] = {0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int r = (tid >> 4) + 8 * u;
                    if (full * kKv8Block + r < n) {
                        float v[8];
                        bf16x8_to_values(*reinterpret_cast<const uint4*>(tails[w] + r * kKv8Dim + (tid & 15) * 8), v);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float m = fabsf(v[k]);
                            if (m < CUDART_INF_F) top[w] = fmaxf(top[w], m);
                        }
                    }
                }
#pragma unroll
            for (int w = 0; w < 2; ++w) {
#pragma unroll
                for (int o = 16; o; o >>= 1) top[w] = fmaxf(top[w], __shfl_xor_sync(0xffffffffu, top[w], o));
                if (lane == 0) ctl->red[w][dw] = top[w];
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kConvThreads) : "memory");
            if (tid < 2) {
                float t = 0.f;
                for (int i = 0; i < kConvWarps; ++i) t = fmaxf(t, ctl->red[tid][i]);
                int e = 0;
                if (t > 0.f) frexpf(t, &e);
                ctl->tail_scale[tid] = exp2f((float)max(min(e - 9, 100), -100));
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kConvThreads) : "memory");
            if (lane == 0) mbar_arrive(bar(&ctl->tail_ready));
        }
        for (int m = 0; m < items && ok; ++m) {
            fetch(m + kRawSlots - 1);
            const int i = tile_of(m), which = which_of(m);
            if (i >= count) continue;
            if (i >= 2) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar(which ? &ctl->v_empty[i & 1] : &ctl->k_empty[i & 1]), ((i >> 1) - 1) & 1, abort_flag));
                if (!ok) break;
            }
            cp_async_wait<kRawSlots - 1>();         // this item has landed
            const int t0 = (j_lo + i) * kWideTile;
            const uint32_t dst = smem_base + (which ? kWVOff : kWKOff) + (i & 1) * kOperand;
            const uint32_t src = raw + (m & (kRawSlots - 1)) * kRawTile;
            const bool masked = t0 + kWideTile > all_see;
            bool bad = false;
            // lanes of the upper 64 dims store their two chunks in the other order: no bank conflicts
            const bool up = ch >= 4;
            const uint32_t d0 = dst + operand_at(row, 2 * ch + (up ? 1 : 0)), d1 = dst + operand_at(row, 2 * ch + (up ? 0 : 1));
            auto put = [&](int u, const uint32_t (&x)[8]) {             // (rows kRowHop apart: the same row & 7)
                const uint32_t at = u * kRowHop * 128;
                st_shared_16(d0 + at, up ? x[4] : x[0], up ? x[5] : x[1], up ? x[6] : x[2], up ? x[7] : x[3]);
                st_shared_16(d1 + at, up ? x[0] : x[4], up ? x[1] : x[5], up ? x[2] : x[6], up ? x[3] : x[7]);
            };
            if (!masked && t0 + kWideTile <= full * kKv8Block) {
#pragma unroll
                for (int u0 = 0; u0 < kConvParts; u0 += 4) {
                    uint4 c[4];
#pragma unroll
                    for (int u = 0; u < 4; ++u) c[u] = ld_shared_16(src + (u0 + u) * kPartBytes);
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        uint32_t x[8];
                        codes_to_half<FMT>(c[u].x, x[0], x[1]);
                        codes_to_half<FMT>(c[u].y, x[2], x[3]);
                        codes_to_half<FMT>(c[u].z, x[4], x[5]);
                        codes_to_half<FMT>(c[u].w, x[6], x[7]);
                        put(u0 + u, x);
                    }
                }
            } else {
#pragma unroll 1
                for (int u = 0; u < kConvParts; ++u) {
                    const int t = t0 + row + kRowHop * u;
                    if (t >= full * kKv8Block && t < (full + 1) * kKv8Block && n % kKv8Block) continue;     // the tail: below
                    uint32_t x[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
                    if (t < full * kKv8Block) {
                        const uint4 c = ld_shared_16(src + u * kPartBytes);
                        codes_to_half<FMT>(c.x, x[0], x[1]);
                        codes_to_half<FMT>(c.y, x[2], x[3]);
                        codes_to_half<FMT>(c.z, x[4], x[5]);
                        codes_to_half<FMT>(c.w, x[6], x[7]);
                        if (FMT == MINF_KV8_E4M3 && which && masked) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) bad |= drop_not_finite(x[k]);
                        }
                    }
                    put(u, x);
                }
            }
            if (has_tail && i == count - 1) {
                const float inv = __fdiv_rn(1.f, ctl->tail_scale[which]);
#pragma unroll 1
                for (int u = 0; u < 8; ++u) {               // (unrolled once: the last tile only)
                    const int r = (tid >> 4) + 8 * u, c16 = tid & 15;
                    uint32_t x[4] = {0u, 0u, 0u, 0u};
                    if (full * kKv8Block + r < n) {
                        float v[8];
                        bf16x8_to_values(*reinterpret_cast<const uint4*>(tails[which] + r * kKv8Dim + c16 * 8), v);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            x[k] = pack_half2_rn(v[2 * k] * inv, v[2 * k + 1] * inv);
                            if (which) bad |= drop_not_finite(x[k]);
                        }
                    }
                    st_shared_16(dst + operand_at(full * kKv8Block - t0 + r, c16), x[0], x[1], x[2], x[3]);
                }
            }
            if (bad) ctl->bad = 1;
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(which ? &ctl->v_full[i & 1] : &ctl->k_full[i & 1]));
        }
        cp_async_wait<0>();
    } else {
        // ------------------------------------------------------------------------------------------- softmax
        const int grp = warp >> 2, r = threadIdx.x & 127, gr = row0 + r;
        const uint32_t t_o = tmem + grp * 256 + ((uint32_t)(32 * (warp & 3)) << 16), t_s = t_o + 128;
        const bool live = gr < a.rows;
        const int lim = live ? all_see + gr % a.n_q : 0;
        const float mul = fabsf(a.scale_log2) * ctl->unit[r];
        const float* ks = a.c.k_scale + bh * (a.c.capacity / kKv8Block);
        const float* vs = a.c.v_scale + bh * (a.c.capacity / kKv8Block);
        float* logits = LOGITS && live ? a.logits + (long long)bh * a.tokens * a.pitch + gr : nullptr;
        const bool warp_live = row0 + 32 * (warp & 3) < a.rows;         // rows behind the last: P of zeros, nothing else
        for (int i = grp; i < count; i += 2) {
            const int t0 = (j_lo + i) * kWideTile;
            float f[2], lv[2], inv_v[2];
            bool tail_half[2];
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int blk = t0 / kKv8Block + x;
                tail_half[x] = blk == full && n % kKv8Block;
                f[x] = blk < full ? ks[blk] : 1.f;
                inv_v[x] = blk < full ? vs[blk] : 1.f;
            }
            if (tail_half[0] || tail_half[1]) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar(&ctl->tail_ready), 0, abort_flag));
                if (!ok) break;
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (tail_half[x]) {
                        f[x] = ctl->tail_scale[0];
                        inv_v[x] = ctl->tail_scale[1];
                    }
            }
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                f[x] *= mul;
                lv[x] = log2f(inv_v[x]);
                inv_v[x] = 1.f / inv_v[x];
            }
            ok = __all_sync(0xffffffffu, mbar_wait(bar(&ctl->s_full[grp]), (i >> 1) & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            if (!warp_live) {
                uint32_t z[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) z[k] = 0u;
                for (int c = 0; c < 4; ++c) tmem_st16(t_s + 16 * c, z);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(bar(&ctl->p_full[grp]));
                continue;
            }
            const bool masked = t0 + kWideTile > all_see;
            const float mx = masked || LOGITS ? row_max<true, LOGITS>(t_s, f, lv, lim - t0, n - t0, LOGITS && logits ? logits + (long long)t0 * a.pitch : nullptr, a.pitch)
                                              : row_max<false, false>(t_s, f, lv, 0, 0, nullptr, 0);
            float alpha = 1.f;
            if (mx > m_ref + 8.f) {                 // the reference is raised on a jump of more than 2^8: P stays far below f16's largest
                alpha = fast_exp2(m_ref - mx);
                l_sum *= alpha;
                m_ref = mx;
            }
            const float ref = m_ref == -CUDART_INF_F ? 0.f : m_ref;
            if (i > 1 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    uint32_t o[32];
                    tmem_ld32(t_o + 32 * c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                    tmem_st32(t_o + 32 * c, o);
                }
            }
            if (masked) row_numerators<true>(t_s, f, lv, inv_v, ref, lim - t0, l_sum);
            else row_numerators<false>(t_s, f, lv, inv_v, ref, 0, l_sum);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bar(&ctl->p_full[grp]));
        }
    }
    // every wait of this kernel ends within its limit: all warps come here
    if (warp < 8) {
        const bool done = mbar_wait(bar(&ctl->o_done), 0, abort_flag);
        ok = __all_sync(0xffffffffu, done && ok);
    }
    __syncthreads();
    if (!ctl->abort) {
        tc_fence_after();
        // join the two groups: the odd tiles' through shared memory (the operands are done with), a column of 128 rows at a time
        float* other = reinterpret_cast<float*>(smem);
        const int r = threadIdx.x & 127, grp = warp >> 2;
        const uint32_t t_o = tmem + (grp & 1) * 256 + ((uint32_t)(32 * (warp & 3)) << 16);
        const bool any = (grp == 0 && count > 0) || (grp == 1 && count > 1);
        const float mine = l_sum == 0.f ? -CUDART_INF_F : (m_ref == -CUDART_INF_F ? l_sum : m_ref + log2f(l_sum));
        if (grp == 1) {
            ctl->lse[r] = mine;
            const float inv = l_sum == 0.f ? 0.f : 1.f / l_sum;
            for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                if (any) {
                    tmem_ld32(t_o + 32 * c, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int k = 0; k < 32; ++k) other[(32 * c + k) * kWideRows + r] = any && l_sum != 0.f ? __uint_as_float(o[k]) * inv : 0.f;
            }
        }
        asm volatile("bar.sync 2, %0;" ::"n"(kWideThreads) : "memory");
        if (grp == 0) {
            const int gr = row0 + r;
            const float theirs = ctl->lse[r], top = fmaxf(mine, theirs);
            const float e0 = mine == -CUDART_INF_F ? 0.f : exp2f(mine - top), e1 = theirs == -CUDART_INF_F ? 0.f : exp2f(theirs - top);
            const float sum = e0 + e1;
            const float w0 = e0 == 0.f ? 0.f : e0 / (sum * l_sum), w1 = e1 == 0.f ? 0.f : e1 / sum;
            const float lse = sum == 0.f ? -CUDART_INF_F : top + log2f(sum);
            const size_t row = bh * a.rows + gr;
            const int hq = h * a.group + gr / a.n_q, t = gr % a.n_q;
            const bool live = gr < a.rows;
            // values left out of the products: from the first tile that not every row sees to its end
            const int bad_lo = max(j_lo, max(all_see, 0) / kWideTile) * kWideTile, bad_hi = min(min(j_hi * kWideTile, n), all_see + t);
            const uint8_t* vc = static_cast<const uint8_t*>(a.c.v) + bh * a.c.capacity * kKv8Dim;
            const __nv_bfloat16* vt = static_cast<const __nv_bfloat16*>(a.c.v_tail) + bh * kKv8Block * kKv8Dim;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
                uint32_t o[32];
                if (any) {
                    tmem_ld32(t_o + 32 * c, o);
                    tmem_wait_ld();
                }
                float x[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                    x[k] = w1 == 0.f ? 0.f : other[(32 * c + k) * kWideRows + r] * w1;
                    if (any && w0 != 0.f) x[k] = fmaf(__uint_as_float(o[k]), w0, x[k]);
                }
                if (!live) continue;
                if (ctl->bad) {
                    for (int tt = bad_lo; tt < bad_hi; ++tt)
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            float v = 0.f;
                            if (tt >= full * kKv8Block) v = __bfloat162float(vt[(tt - full * kKv8Block) * kKv8Dim + 32 * c + k]);
                            else if (FMT == MINF_KV8_E4M3 && (vc[(size_t)tt * kKv8Dim + 32 * c + k] & 0x7f) == 0x7f) v = CUDART_NAN_F;
                            if (!(fabsf(v) < CUDART_INF_F)) x[k] += v;
                        }
                }
                if (a.splits > 1) {
                    float4* dst = reinterpret_cast<float4*>(a.part_o + (row * a.splits + split) * kKv8Dim + 32 * c);
#pragma unroll
                    for (int k = 0; k < 8; ++k) dst[k] = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
                } else {
                    uint2* dst = reinterpret_cast<uint2*>(a.o + b * a.os[0] + hq * a.os[1] + t * a.os[2] + 32 * c);
#pragma unroll
                    for (int k = 0; k < 8; ++k) dst[k] = make_uint2(pack_bf16x2(x[4 * k], x[4 * k + 1]), pack_bf16x2(x[4 * k + 2], x[4 * k + 3]));
                }
            }
            if (live) {
                if (a.splits > 1) {
                    a.part_lse[row * a.splits + split] = lse;
                } else {
                    if (a.lse) a.lse[((size_t)b * a.c.heads * a.group + hq) * a.n_q + t] = lse;
                    if (a.row_lse) a.row_lse[row] = lse;
                }
            }
        }
    } else {
        // a wait was abandoned: give the copies and products in flight time to land before shared memory and TMEM go on
        __nanosleep(50000);
        if (threadIdx.x == 0) atomicOr(a.c.status + MINF_ST_ERROR, 1);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <int FMT, bool LOGITS>
static cudaError_t launch_wide(const Kv8AttnArgs& a, int tiles, cudaStream_t stream) {
    constexpr int bytes = kWCtlOff + sizeof(WideCtl);
    const cudaError_t e = cudaFuncSetAttribute(kv8_attention_wide_kernel<FMT, LOGITS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return e;
    kv8_attention_wide_kernel<FMT, LOGITS><<<dim3(a.splits, a.c.heads * tiles, a.c.batch), kWideThreads, bytes, stream>>>(a, tiles);
    return cudaGetLastError();
}

cudaError_t launch_attention_wide(const Kv8AttnArgs& a, int tiles, cudaStream_t stream) {
    if (a.c.format == MINF_KV8_E4M3) return a.logits ? launch_wide<MINF_KV8_E4M3, true>(a, tiles, stream) : launch_wide<MINF_KV8_E4M3, false>(a, tiles, stream);
    return a.logits ? launch_wide<MINF_KV8_INT8, true>(a, tiles, stream) : launch_wide<MINF_KV8_INT8, false>(a, tiles, stream);
}

}  // namespace minf
