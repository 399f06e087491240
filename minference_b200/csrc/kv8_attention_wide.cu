// Attention over an 8-bit cache for many query rows per cache head (several new tokens, large groups): the formulas and
// the splitting of kv8_attention.cu, on the tcgen05 tensor cores.
//
// One CTA owns 128 rows of a head and a stretch of its tokens, in tiles of 128.  Warp roles:
//   warps 0-3, 4-7       softmax of the even / odd tiles, a thread per row.  Each group keeps its own maximum, sum and output
//                        (O and S in TMEM, P written over S as f16), so that the loads and exchanges of one tile run under
//                        the exponentials of the other; the two results are joined at the end
//   warps 8-10, 11-13    turn codes into f16 operands, one team the keys', one the values': cp.async into two 16 KB tiles,
//                        the next one in flight while one is converted into the team's two 128-byte-swizzled stages.  A
//                        thread converts what it copied itself, so the copies need no barrier
//   warp 14              issues the MMAs
// (Four warps share a scheduler at most, so of the launch's registers a thread has 128: half a row of S, and 88 bytes of spills,
// 96 with logits.  Moving registers to the softmax warps, as the prefill kernel of this library does, was not tried.)  Built and measured as well:
// two threads a row and one group (3070 cycles a tile, all of it one chain), conversion by one team of four warps (its
// 2200 cycles a tile bound the rest).
// TMEM: O and S of the two groups, 4 x 128 columns.
//
// The tail's bf16 values become f16 by a power of two for the block (what is lost lies 2^-33 below its largest value).
// In tiles that some row does not see to its end, values that are infinite or NaN are left out of the product (zero
// times them would reach rows that do not see them) and added to the rows that do at the end.
//
// Bound: the chain of a softmax warp.  A tile takes 2400 cycles (131072 tokens of 8 heads: 128 rows 96 us, 256 rows 162 us;
// 256 new tokens of 32 heads over 16384: 101 us), of which the products need 1024, the exponentials 1024, shared memory 1792
// and HBM's share 1400; ALU 58 % busy, issue slots 55 %, exponentials 43 %, tensor pipe 41 %.  Two ways round a part of it were
// 2-4 % slower: S in two halves, the next one asked for as soon as P of the half before is used up; codes straight from HBM
// into registers instead of through the raw tiles.
#include "kv8_attention.cuh"

#include <math_constants.h>

#include "sm100_ptx.cuh"

namespace minf {

constexpr int kWideTile = 128;                      // tokens of a tile
constexpr uint32_t kOperand = 128 * 256;            // 128 rows x 128 f16
constexpr uint32_t kRawTile = 128 * 128;            // codes of a tile
constexpr int kRawSlots = 2;                        // per team
constexpr uint32_t kWQOff = 0, kWKOff = kOperand, kWVOff = 3 * kOperand, kWRawOff = 5 * kOperand;
constexpr uint32_t kWCtlOff = kWRawOff + 2 * kRawSlots * kRawTile;
constexpr int kConvWarps = 3, kMmaWarp = 8 + 2 * kConvWarps;
constexpr int kWideThreads = (kMmaWarp + 1) * 32;
constexpr int kConvThreads = kConvWarps * 32;
constexpr int kRowHop = kConvThreads / 8;                      // rows that a team takes at a time
constexpr int kConvParts = (128 + kRowHop - 1) / kRowHop;      // 16-byte pieces of a tile a thread converts (the last one: some threads)
static_assert(kRowHop % 4 == 0 && kRowHop % 8 != 0, "rows kRowHop apart differ in bit 2 of r & 7");

struct WideCtl {
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_half[2][2], tail_ready, o_done;
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
            mbar_init(bar(&ctl->p_half[s][0]), 128);    // the rows' threads
            mbar_init(bar(&ctl->p_half[s][1]), 128);
        }
        mbar_init(bar(&ctl->tail_ready), 2 * kConvWarps);
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
        const uint4* q = r < a.rows ? reinterpret_cast<const uint4*>(a.q + b * a.qs[0] + (long long)(h * a.group + r / a.n_q) * a.qs[1] + (long long)(r % a.n_q) * a.qs[2]) : nullptr;
        uint4 x[16];
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = q ? q[i] : make_uint4(0u, 0u, 0u, 0u);
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
        e = max(e - 8, -126);
        const float inv = __uint_as_float(((uint32_t)(127 - e) << 23) | (a.scale_log2 < 0.f ? 0x80000000u : 0u));
        ctl->unit[threadIdx.x] = __uint_as_float((uint32_t)(127 + e) << 23);
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
            constexpr uint32_t idesc = umma_idesc(128, 128, false, false, true);
            const uint32_t d = tmem + (i & 1) * 256, p = d + 128;
            const uint32_t v_lo = ((smem_base + kWVOff + (i & 1) * kOperand) >> 4) | ((16384u >> 4) << 16);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                ok = ok && wait(&ctl->p_half[i & 1][half], (i >> 1) & 1);
                if (!ok) return;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int kk = 4 * half; kk < 4 * half + 4; ++kk)
                        umma_ts(d, p + kk * 8, desc(v_lo + kk * (2048 >> 4)), idesc, (i > 1 || kk > 0) ? 1u : 0u);
                    if (half) umma_commit(bar(&ctl->v_empty[i & 1]));
                }
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
        const int which = warp >= 8 + kConvWarps, dw = (warp - 8) % kConvWarps, tid = threadIdx.x - 256 - which * kConvThreads;
        const uint8_t* codes = static_cast<const uint8_t*>(which ? a.c.v : a.c.k) + bh * a.c.capacity * kKv8Dim;
        const __nv_bfloat16* tail = static_cast<const __nv_bfloat16*>(which ? a.c.v_tail : a.c.k_tail) + bh * kKv8Block * kKv8Dim;
        constexpr int kPartBytes = kConvThreads * 16;
        // Rows row + kRowHop u, 16 codes from 16 ch.  Eight neighbouring lanes have chunks 0-3 of a row and 4-7 of its
        // neighbour: so their operand chunks lie in different banks (the upper 64 dims lie 16 KB behind the lower).
        const int quad = (tid >> 2) & 3;
        const int row = (tid >> 4) * 2 + (quad == 1 || quad == 2), ch = (tid & 3) + 4 * (quad & 1);
        const uint32_t mine = row * 128 + ch * 16, raw = smem_base + kWRawOff + which * kRawSlots * kRawTile + mine;
        unsigned long long* const full_bar = which ? ctl->v_full : ctl->k_full;
        unsigned long long* const empty_bar = which ? ctl->v_empty : ctl->k_empty;
        auto fetch = [&](int i) {
            if (i < count) {
                const int t0 = (j_lo + i) * kWideTile;
                const uint8_t* src = codes + (size_t)t0 * kKv8Dim + mine;
                const uint32_t dst = raw + (i & 1) * kRawTile;
                const int rows = min(full * kKv8Block - t0, kWideTile) - row;       // rows of complete blocks from this thread's on
#pragma unroll
                for (int u = 0; u < kConvParts; ++u)
                    if (kRowHop * u < rows) cp_async_16(dst + u * kPartBytes, src + u * kPartBytes);
            }
            cp_async_commit();
        };
        fetch(0);
        fetch(1);
        if (has_tail) {                             // the tail's scale, before its tile is due
            float top = 0.f;
#pragma unroll 4
            for (int r = tid >> 4; r < kKv8Block; r += kConvThreads / 16) {
                if (full * kKv8Block + r < n) {
                    float v[8];
                    bf16x8_to_values(*reinterpret_cast<const uint4*>(tail + r * kKv8Dim + (tid & 15) * 8), v);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float m = fabsf(v[k]);
                        if (m < CUDART_INF_F) top = fmaxf(top, m);
                    }
                }
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (lane == 0) ctl->red[which][dw] = top;
            asm volatile("bar.sync %0, %1;" ::"r"(1 + which), "n"(kConvThreads) : "memory");
            if (tid == 0) {
                float t = 0.f;
                for (int i = 0; i < kConvWarps; ++i) t = fmaxf(t, ctl->red[which][i]);
                int e = 0;
                if (t > 0.f) frexpf(t, &e);
                ctl->tail_scale[which] = __uint_as_float((uint32_t)(127 + max(e - 9, -126)) << 23);
            }
            asm volatile("bar.sync %0, %1;" ::"r"(1 + which), "n"(kConvThreads) : "memory");
            if (lane == 0) mbar_arrive(bar(&ctl->tail_ready));
        }
#pragma unroll 1
        for (int i = 0; i < count; ++i) {
            cp_async_wait<1>();                     // this tile has landed
            const int t0 = (j_lo + i) * kWideTile;
            const uint32_t src = raw + (i & 1) * kRawTile, dst = smem_base + (which ? kWVOff : kWKOff) + (i & 1) * kOperand;
            uint4 c[kConvParts];
#pragma unroll
            for (int u = 0; u < kConvParts; ++u)
                c[u] = u < kConvParts - 1 || row + kRowHop * u < kWideTile ? ld_shared_16(src + u * kPartBytes) : make_uint4(0u, 0u, 0u, 0u);
            if (i >= 2) {
                ok = __all_sync(0xffffffffu, mbar_wait(bar(&empty_bar[i & 1]), ((i >> 1) - 1) & 1, abort_flag));
                if (!ok) break;
            }
            const bool masked = t0 + kWideTile > all_see;
            bool bad = false;
            // rows kRowHop apart differ in bit 2 of r & 7, which the chunks' places are xored with: 64 bytes on or back
            const uint32_t d0 = dst + operand_at(row, 2 * ch), d1 = dst + operand_at(row, 2 * ch + 1);
            auto put = [&](int u, const uint32_t (&x)[8]) {
                const uint32_t at = u * kRowHop * 128, flip = (u & 1) * 64;
                if (u < kConvParts - 1 || row + kRowHop * u < kWideTile) {
                    st_shared_16((d0 ^ flip) + at, x[0], x[1], x[2], x[3]);
                    st_shared_16((d1 ^ flip) + at, x[4], x[5], x[6], x[7]);
                }
            };
            auto halves = [&](const uint4& w, uint32_t (&x)[8]) {
                codes_to_half<FMT>(w.x, x[0], x[1]);
                codes_to_half<FMT>(w.y, x[2], x[3]);
                codes_to_half<FMT>(w.z, x[4], x[5]);
                codes_to_half<FMT>(w.w, x[6], x[7]);
            };
            // Shared memory is read in order: once the last pieces are used, all are in registers, and the next tile but one may
            // be copied over them.
            if (!masked && t0 + kWideTile <= full * kKv8Block) {
#pragma unroll
                for (int u = kConvParts - 1; u >= 0; --u) {
                    uint32_t x[8];
                    halves(c[u], x);
                    put(u, x);
                    if (u == kConvParts - 2) fetch(i + 2);
                }
            } else {
#pragma unroll
                for (int u = kConvParts - 1; u >= 0; --u) {
                    const int t = t0 + row + kRowHop * u;
                    uint32_t x[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
                    if (t < full * kKv8Block) {
                        halves(c[u], x);
                        if (FMT == MINF_KV8_E4M3 && which && masked) {
#pragma unroll
                            for (int k = 0; k < 8; ++k) bad |= drop_not_finite(x[k]);
                        }
                    }
                    if (t < full * kKv8Block || t >= (full + 1) * kKv8Block || n % kKv8Block == 0) put(u, x);      // the tail: below
                }
            }
            if (masked || t0 + kWideTile > full * kKv8Block) fetch(i + 2);
            if (has_tail && i == count - 1) {
                const float inv = __fdiv_rn(1.f, ctl->tail_scale[which]);
#pragma unroll 1
                for (int r = tid >> 4; r < kKv8Block; r += kConvThreads / 16) {
                    const int c16 = tid & 15;
                    uint32_t x[4] = {0u, 0u, 0u, 0u};
                    if (full * kKv8Block + r < n) {
                        float v[8];
                        bf16x8_to_values(*reinterpret_cast<const uint4*>(tail + r * kKv8Dim + c16 * 8), v);
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
            if (lane == 0) mbar_arrive(bar(&full_bar[i & 1]));
        }
        cp_async_wait<0>();
    } else {
        // ------------------------------------------------------------------------------------------- softmax
        const int grp = warp >> 2, r = threadIdx.x & 127, gr = row0 + r;
        const uint32_t t_o = tmem + grp * 256 + ((uint32_t)(32 * (warp & 3)) << 16), t_s = t_o + 128;
        const bool live = gr < a.rows;
        const int lim = live ? all_see + gr % a.n_q : 0x7fffffff;      // (rows behind the last: anything, they are dropped)
        const float mul = fabsf(a.scale_log2) * ctl->unit[r];
        const float* ks = a.c.k_scale + bh * (a.c.capacity / kKv8Block);
        const float* vs = a.c.v_scale + bh * (a.c.capacity / kKv8Block);
        float* logits = LOGITS && live ? a.logits + (long long)bh * a.tokens * a.pitch + gr : nullptr;
        const bool warp_live = row0 + 32 * (warp & 3) < a.rows;         // rows behind the last: P of zeros, nothing else
        float next_k[2], next_v[2];
        auto scales = [&](int i) {                  // of a tile's two blocks, read a turn ahead
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int blk = (j_lo + i) * 2 + x;
                const bool there = i < count && blk < full;
                next_k[x] = there ? ks[blk] : 1.f;
                next_v[x] = there ? vs[blk] : 1.f;
            }
        };
        scales(grp);
        for (int i = grp; i < count; i += 2) {
            const int t0 = (j_lo + i) * kWideTile;
            float f[2] = {next_k[0], next_k[1]}, inv_v[2] = {next_v[0], next_v[1]}, lv[2];
            if (t0 + kWideTile > full * kKv8Block && n % kKv8Block) {   // the tail is one of the blocks
                ok = __all_sync(0xffffffffu, mbar_wait(bar(&ctl->tail_ready), 0, abort_flag));
                if (!ok) break;
                const int x = full & 1;
                f[0] = x == 0 ? ctl->tail_scale[0] : f[0];
                f[1] = x == 1 ? ctl->tail_scale[0] : f[1];
                inv_v[0] = x == 0 ? ctl->tail_scale[1] : inv_v[0];
                inv_v[1] = x == 1 ? ctl->tail_scale[1] : inv_v[1];
            }
            scales(i + 2);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                f[x] *= mul;
                lv[x] = __log2f(inv_v[x]);
                inv_v[x] = __fdividef(kHeadroomOut, inv_v[x]);
            }
            ok = __all_sync(0xffffffffu, mbar_wait(bar(&ctl->s_full[grp]), (i >> 1) & 1, abort_flag));
            if (!ok) break;
            tc_fence_after();
            if (!warp_live) {
                uint32_t z[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) z[k] = 0u;
#pragma unroll 1
                for (int c = 0; c < 8; ++c) tmem_st8(t_s + 8 * c, z);
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(bar(&ctl->p_half[grp][0]));
                mbar_arrive(bar(&ctl->p_half[grp][1]));
                continue;
            }
            const int seen = lim - t0;              // of this tile's tokens
            // Columns 32 c .. of S, -inf where the row does not see the token.
            auto hide = [&](int c, uint32_t (&x)[32]) {
                const int left = seen - 32 * c;
                if (left < 32) {
                    const uint32_t cm = left <= 0 ? 0u : (1u << left) - 1u;
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (!((cm >> k) & 1u)) x[k] = 0xff800000u;
                }
            };
            auto largest = [&](const uint32_t (&x)[32]) {
                float m4[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
                for (int k = 0; k < 32; k += 2) m4[(k >> 1) & 3] = max3(m4[(k >> 1) & 3], __uint_as_float(x[k]), __uint_as_float(x[k + 1]));
                return fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
            };
            // The maximum first, of the second block and then of the first, which stays in registers: its P goes over the
            // columns it came from, and is on the tensor cores while the second block is read again.
            uint32_t s0[32], s1[32];
            tmem_ld32(t_s + 64, s0);
            tmem_ld32(t_s + 96, s1);
            tmem_wait_ld();
            hide(2, s0);
            float mb = largest(s0);
            tmem_ld32(t_s, s0);
            hide(3, s1);
            mb = fmaxf(mb, largest(s1));
            tmem_ld32(t_s + 32, s1);
            tmem_wait_ld();
            hide(0, s0);
            hide(1, s1);
            const float ma = fmaxf(largest(s0), largest(s1));
            const float mx = fmaxf(ma == -CUDART_INF_F ? ma : fmaf(ma, f[0], lv[0]), mb == -CUDART_INF_F ? mb : fmaf(mb, f[1], lv[1]));   // (-inf times zero)
            float alpha = 1.f;
            if (mx > m_ref + 8.f) {                 // the reference is raised on a jump of more than 2^8: P stays below f16's largest
                alpha = fast_exp2(m_ref - mx);
                l_sum *= alpha;
                m_ref = mx;
            }
            const float ref = m_ref == -CUDART_INF_F ? 0.f : m_ref - kHeadroom;
            if (i > 1 && __any_sync(0xffffffffu, alpha != 1.f)) {       // (O is at rest: this tile's S came behind its last product)
#pragma unroll 1
                for (int c = 0; c < 16; ++c) {
                    uint32_t o[8];
                    tmem_ld8(t_o + 8 * c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 8; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                    tmem_st8(t_o + 8 * c, o);
                }
            }
            // P of 32 tokens of block x, columns 32 c of S; the sum of the numerators
            auto numerators = [&](int c, int x, uint32_t (&sc)[32]) {
                if (LOGITS && logits) {
                    float* to = logits + (long long)(t0 + 32 * c) * a.pitch;
                    if (t0 + kWideTile <= min(n, lim)) {
#pragma unroll
                        for (int k = 0; k < 32; ++k, to += a.pitch) *to = __uint_as_float(sc[k]) * f[x];
                    } else {
#pragma unroll
                        for (int k = 0; k < 32; ++k, to += a.pitch)
                            if (t0 + 32 * c + k < n) *to = 32 * c + k < seen ? __uint_as_float(sc[k]) * f[x] : -CUDART_INF_F;
                    }
                }
                const float d = lv[x] - ref;
                const uint64_t f2 = pack_f32x2(f[x], f[x]), d2 = pack_f32x2(d, d);
                uint64_t sum2[2] = {0ull, 0ull};
                const bool zero = f[x] == 0.f && seen < 32 * c + 32;    // (the only masked logits the product would not leave at -inf)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    uint32_t p[8];
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const int kk = 16 * hf + k;
                        float x0, x1;
                        unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(sc[kk]), __uint_as_float(sc[kk + 1])), f2, d2), x0, x1);
                        x0 = fast_exp2(x0);
                        x1 = fast_exp2(x1);
                        if (zero) {
                            if (32 * c + kk >= seen) x0 = 0.f;
                            if (32 * c + kk + 1 >= seen) x1 = 0.f;
                        }
                        sum2[(k >> 1) & 1] = add_f32x2(sum2[(k >> 1) & 1], pack_f32x2(x0, x1));
                        p[k >> 1] = pack_half2_rn(x0, x1);
                    }
                    tmem_st8(t_s + 16 * c + 8 * hf, p);
                }
                float a0, a1;
                unpack_f32x2(add_f32x2(sum2[0], sum2[1]), a0, a1);
                return a0 + a1;
            };
            float sum = numerators(0, 0, s0);
            tmem_ld32(t_s + 64, s0);
            sum += numerators(1, 0, s1);
            l_sum = fmaf(sum, inv_v[0], l_sum);
            tmem_wait_ld();
            tmem_ld32(t_s + 96, s1);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bar(&ctl->p_half[grp][0]));
            hide(2, s0);
            sum = numerators(2, 1, s0);
            tmem_wait_ld();
            hide(3, s1);
            sum += numerators(3, 1, s1);
            l_sum = fmaf(sum, inv_v[1], l_sum);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(bar(&ctl->p_half[grp][1]));
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
            const float inv = l_sum == 0.f ? 0.f : kHeadroomOut / l_sum;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
                uint32_t o[16];
                if (any) {
                    tmem_ld16(t_o + 16 * c, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int k = 0; k < 16; ++k) other[(16 * c + k) * kWideRows + r] = any && l_sum != 0.f ? __uint_as_float(o[k]) * inv : 0.f;
            }
        }
        __syncthreads();
        if (grp == 0) {
            const int gr = row0 + r;
            const float theirs = ctl->lse[r], top = fmaxf(mine, theirs);
            const float e0 = mine == -CUDART_INF_F ? 0.f : exp2f(mine - top), e1 = theirs == -CUDART_INF_F ? 0.f : exp2f(theirs - top);
            const float sum = e0 + e1;
            const float w0 = e0 == 0.f ? 0.f : e0 * kHeadroomOut / (sum * l_sum), w1 = e1 == 0.f ? 0.f : e1 / sum;
            const float lse = sum == 0.f ? -CUDART_INF_F : top + log2f(sum);
            const size_t row = bh * a.rows + gr;
            const int hq = h * a.group + gr / a.n_q, t = gr % a.n_q;
            const bool live = gr < a.rows;
            // values left out of the products: from the first tile that not every row sees to its end
            const int bad_lo = max(j_lo, max(all_see, 0) / kWideTile) * kWideTile, bad_hi = min(min(j_hi * kWideTile, n), all_see + t);
            const uint8_t* vc = static_cast<const uint8_t*>(a.c.v) + bh * a.c.capacity * kKv8Dim;
            const __nv_bfloat16* vt = static_cast<const __nv_bfloat16*>(a.c.v_tail) + bh * kKv8Block * kKv8Dim;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
                __syncwarp();                       // (a warp's rows part below; its loads from TMEM are of all lanes together)
                uint32_t o[16];
                if (any) {
                    tmem_ld16(t_o + 16 * c, o);
                    tmem_wait_ld();
                }
                float x[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    x[k] = w1 == 0.f ? 0.f : other[(16 * c + k) * kWideRows + r] * w1;
                    if (any && w0 != 0.f) x[k] = fmaf(__uint_as_float(o[k]), w0, x[k]);
                }
                if (!live) continue;
                const int d = 16 * c;
                if (ctl->bad) {
                    for (int tt = bad_lo; tt < bad_hi; ++tt)
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            float v = 0.f;
                            if (tt >= full * kKv8Block) v = __bfloat162float(vt[(tt - full * kKv8Block) * kKv8Dim + d + k]);
                            else if (FMT == MINF_KV8_E4M3 && (vc[(size_t)tt * kKv8Dim + d + k] & 0x7f) == 0x7f) v = CUDART_NAN_F;
                            if (!(fabsf(v) < CUDART_INF_F)) x[k] += v;
                        }
                }
                if (a.splits > 1) {
                    float4* dst = reinterpret_cast<float4*>(a.part_o + (row * a.splits + split) * kKv8Dim + d);
#pragma unroll
                    for (int k = 0; k < 4; ++k) dst[k] = make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
                } else {
                    uint2* dst = reinterpret_cast<uint2*>(a.o + b * a.os[0] + hq * a.os[1] + t * a.os[2] + d);
#pragma unroll
                    for (int k = 0; k < 4; ++k) dst[k] = make_uint2(pack_bf16x2(x[4 * k], x[4 * k + 1]), pack_bf16x2(x[4 * k + 2], x[4 * k + 3]));
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
    static std::atomic<unsigned long long> allowed{0};
    const cudaError_t e = allow_shared(kv8_attention_wide_kernel<FMT, LOGITS>, bytes, allowed);
    if (e != cudaSuccess) return e;
    kv8_attention_wide_kernel<FMT, LOGITS><<<dim3(a.splits, a.c.heads * tiles, a.c.batch), kWideThreads, bytes, stream>>>(a, tiles);
    return cudaGetLastError();
}

cudaError_t launch_attention_wide(const Kv8AttnArgs& a, int tiles, cudaStream_t stream) {
    if (a.c.format == MINF_KV8_E4M3) return a.logits ? launch_wide<MINF_KV8_E4M3, true>(a, tiles, stream) : launch_wide<MINF_KV8_E4M3, false>(a, tiles, stream);
    return a.logits ? launch_wide<MINF_KV8_INT8, true>(a, tiles, stream) : launch_wide<MINF_KV8_INT8, false>(a, tiles, stream);
}

}  // namespace minf
