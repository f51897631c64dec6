// tsb_cache_prompt.cuh - attention of many queries over the 8-bit cache on tcgen05 (16-bit queries): part of tsb_cache.cu.
//
// CTA (tile of 128 rows, key / value head, request); rows are query tokens times the heads of the group, so a grouped model
// reads a key for all of them.  Keys and values in tiles of kN tokens, two stages each:
//   warps 0-7   softmax: two threads a row (a tensor-memory lane), half of a tile's columns each, who meet for the row's
//               maximum; scores from tensor memory, weights back to it as fp16
//   warps 8-15  the codes from the cache to fp16 operands in shared memory (exact: the product needs 16-bit operands, and
//               int8 products would take three planes of the queries and three tensor-memory reads a score)
//   warp 16     issues the products (one lane): S = Q K^T (both K-major), O += P V (P in tensor memory, V as it lies, its
//               value columns contiguous: MN-major)
// S and P are double buffered, so the products of tile j + 1 and j - 1 run while tile j is in the softmax.  O stays in tensor
// memory; its rows are rescaled only when a row's score exceeds its reference by 2^4 (or a block's value scale the
// largest so far), which after a row's first tiles is rare.
// Weights are exp2(x - reference + 11), at most 2^15, times the block's value scale relative to the largest so far: fp16 keeps
// 11 bits of those down to 2^-25 of the reference, and for fp16 outputs (LO), whose own rounding is no coarser, a second fp16
// value holds the rest.  The sums l and everything of the softmax are fp32.
// What bounds it: a tile's way from scores to weights, two passes over tensor memory (3300 cycles a tile of 64 keys at head_dim 256, the
// products 1411 of them).  2048 queries over 8192 keys, 16 heads of 256: 403 us, 597 TFLOP/s, 256 tiles in two waves.
#pragma once

#include <type_traits>

#include "tsb_tc.cuh"

namespace tsb {
namespace {

constexpr unsigned kSitePrompt = 0xC0000001u;   // the error word when a wait of this kernel gave up
constexpr int kPromptThreads = 17 * 32, kConvThreads = 8 * 32, kMmaWarp = 16;
constexpr float kRefShift = 11.0f, kRefLazy = 4.0f;

template <int D, bool LO>
struct Prompt {
    static constexpr int kN = D == 256 || LO ? 64 : 128;
    static constexpr int kQ = 128 * D * 2, kKV = kN * D * 2;
    static constexpr int kGroups = kN / 16;
    // tensor memory columns: O, S twice, P twice (two weights a column), with LO the weights' low halves twice
    static constexpr int kS = D, kP = D + 2 * kN, kLow = kP + kN;
    static_assert(kP + (LO ? 2 : 1) * kN <= 512, "tensor memory");
    static constexpr int kSmem = kQ + 4 * kKV + 1024;                      // and room to align
    static constexpr int kAsk = kSmem > 120 * 1024 ? kSmem : 120 * 1024;   // one CTA a SM: each takes all of tensor memory
};
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr, int chunk_bytes) {   // MN-major, 128-byte swizzle
    return (uint64_t) ((addr >> 4) & 0x3FFFu) | ((uint64_t) (chunk_bytes >> 4) << 16) | ((uint64_t) (1024 >> 4) << 32) |
           ((uint64_t) 1 << 46) | ((uint64_t) 2 << 61);
}
// Issued by one lane of the (converged) calling warp.  The whole warp walks the product loop, so that descriptors and
// addresses stay in uniform registers: under a single lane's branch the same loop spent 3000 cycles a tile on issuing 20
// products.
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n .reg .pred p, e;\n elect.sync _|e, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
                 " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {      // by the lane that issued (elect.sync picks the same one)
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
                 : "memory");
}
#define TSB_R8(x, o) "=r"(x[o]), "=r"(x[o + 1]), "=r"(x[o + 2]), "=r"(x[o + 3]), "=r"(x[o + 4]), "=r"(x[o + 5]), "=r"(x[o + 6]), "=r"(x[o + 7])
#define TSB_W8(x, o) "r"(x[o]), "r"(x[o + 1]), "r"(x[o + 2]), "r"(x[o + 3]), "r"(x[o + 4]), "r"(x[o + 5]), "r"(x[o + 6]), "r"(x[o + 7])
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : TSB_R8(r, 0), TSB_R8(r, 8), TSB_R8(r, 16), TSB_R8(r, 24)
                 : "r"(addr));
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : TSB_R8(r, 0), TSB_R8(r, 8)
                 : "r"(addr));
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::TSB_W8(r, 0),
                 TSB_W8(r, 8), "r"(addr)
                 : "memory");
}
#undef TSB_R8
#undef TSB_W8
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Four codes in order as two pairs of fp16.
__device__ __forceinline__ void codes4(uint32_t w, uint32_t& a, uint32_t& b) {
    constexpr uint32_t bias = 0x64806480u;
    const uint32_t x = w ^ 0x80808080u;
    a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 u = __hsub2(*(const __half2*) &a, *(const __half2*) &bias), v = __hsub2(*(const __half2*) &b, *(const __half2*) &bias);
    a = *(const uint32_t*) &u, b = *(const uint32_t*) &v;
}

template <int D, bool LO>
__global__ void __launch_bounds__(kPromptThreads, 1) k_attn_prompt(const __grid_constant__ AttnParams p) {
    using P = Prompt<D, LO>;
    constexpr int N = P::kN, NG = P::kGroups, CH = D / 16;       // CH: 16-code chunks of a token
    extern __shared__ __align__(1024) uint8_t prompt_smem[];
    uint8_t* smem = prompt_smem + ((1024 - (smem_u32(prompt_smem) & 1023)) & 1023);
    __shared__ uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], s_free[2], p_full[2], pv_done[2], drained;
    __shared__ uint32_t tbase;
    __shared__ float rowf[128], meet[2][2][128], sums[2][128];
    __shared__ float heads[4][3][NG];                             // key scales, value scales, whether the block is in the cache
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rt = gridDim.x - 1 - blockIdx.x, h = blockIdx.y, r = blockIdx.z;
    const Req q = attn_req(p, r);
    const int rows = q.n * p.G;
    if (rt == 0 && h == 0 && tid == 0) check_request(p, r);
    if (rt * 128 >= rows) return;
    int first, steps;
    tile_steps<128>(p, q, rt, first, steps);
    const int t_first = first * kStep, t_end = (first + steps) * kStep, n = (steps * kStep + N - 1) / N;
    uint8_t *qs = smem, *ks = smem + P::kQ, *vs = ks + 2 * P::kKV;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 8), mbar_init(&k_empty[i], 1), mbar_init(&v_full[i], 8), mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 2), mbar_init(&s_free[i], 8), mbar_init(&p_full[i], 8), mbar_init(&pv_done[i], 1);
        }
        mbar_init(&drained, 1);
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tbase)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // the rows, scaled by a power of two to [2^10, 2^11) at their largest: exact in fp16 down to 2^-35 of it
    for (int i = warp; i < 128; i += 17) {
        const int row = rt * 128 + i;
        float x[D / 32], peak = 0.0f;
        bool nan = false;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            x[j] = row < rows ? load_elem(p.q, (int64_t) (q.tok + row / p.G) * p.q_tok + (int64_t) (h * p.G + row % p.G) * p.q_head + j * 32 + lane, p.type) : 0.0f;
            peak = fmaxf(peak, fabsf(x[j])), nan |= !(fabsf(x[j]) <= 3.4028235e38f);
        }
        peak = warp_max(peak);
        nan = __any_sync(0xffffffffu, nan);
        const int e = min(max((int) (__float_as_uint(peak) >> 23) & 255, 11), 254);
        const float up = copysignf(__uint_as_float((uint32_t) min(264 - e, 254) << 23), p.scale_log2);
        const float back = __uint_as_float((uint32_t) max(e - 10, 1) << 23);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            const int d = j * 32 + lane;
            *(__half*) (qs + (d >> 6) * 16384 + sw128(i, (d & 63) >> 3) + (d & 7) * 2) = __float2half_rn(nan ? 0.0f : x[j] * up);
        }
        if (lane == 0) rowf[i] = nan ? __uint_as_float(0x7fffffffu) : fabsf(p.scale_log2) * back;
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tbase;

    if (warp < 8) {
        // ------------------------------------------------------------------------------------------------ softmax
        constexpr int NH = N / 2, DH = D / 2;                     // a thread's columns of scores and of outputs
        const int wq = warp & 3, half = warp >> 2;
        const uint32_t mine = tmem + ((uint32_t) (wq * 32) << 16);
        const int i = wq * 32 + lane, row = rt * 128 + i;
        const int pos = max(q.len - q.n + min(row, rows - 1) / p.G, -1);   // -1: no keys
        const int pmin = q.len - q.n + (rt * 128) / p.G;
        const int lmax = p.window > 0 ? window_first(p, q, (min(rt * 128 + 128, rows) - 1) / p.G) : INT_MIN;
        const int win = p.window > 0 ? p.window : INT_MAX;
        const float rf = rowf[i];
        float m = -INFINITY, l = 0.0f, ref = 0.0f, per_ref = 0.0f;
        bool ok = true;
        // a wait that gave up ends the waiting, not the loop: a row's two warps meet at every barrier
        auto wait = [&](uint64_t* bar, int j) {
            if (ok) ok = mbar_wait_bounded(bar, (j >> 1) & 1, p.err, kSitePrompt);
            ok = __all_sync(0xffffffffu, ok);
        };
        for (int j = 0; j < n; ++j) {
            const int b = j & 1, t0 = t_first + j * N;
            wait(&s_full[b], j);
            tc_fence_after();
            const float(*hd)[NG] = heads[j & 3];
            // columns that the row sees: a range, less the groups outside the cache
            bool all = !(t0 + N - 1 > pmin || t0 < lmax || t0 + N > t_end);
            float top = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) all &= hd[2][g] != 0.0f, top = fmaxf(top, hd[1][g]);
            const int c_hi = pos - t0, c_lo = pos - win >= t0 ? pos - win - t0 + 1 : 0;
            auto seen = [&](int c0) -> uint32_t {                 // bits of columns c0 .. c0 + 31
                const int hi = c_hi - c0, lo = c_lo - c0;
                uint32_t v = hi < 0 ? 0u : hi >= 31 ? ~0u : (2u << hi) - 1;
                if (lo > 0) v &= lo > 31 ? 0u : ~0u << lo;
                if (hd[2][c0 / 16] == 0.0f) v &= 0xffff0000u;
                if (hd[2][c0 / 16 + 1] == 0.0f) v &= 0x0000ffffu;
                return v;
            };
            const uint32_t from = mine + P::kS + b * N + half * NH;
            float mx = -INFINITY;
            uint32_t s[32];                                       // the last 32 columns stay for the weights
            uint32_t see = 0;
#pragma unroll 1
            for (int c0 = 0; c0 < NH; c0 += 32) {
                const int ca = half * NH + c0;
                tm_ld32(from + c0, s);
                const float sc[2] = {hd[0][ca / 16] * rf, hd[0][ca / 16 + 1] * rf};
                tmem_wait_ld();
                if (!all) {
                    see = seen(ca);
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (!(see >> c & 1)) s[c] = 0xff800000u;
                }
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    float y = __uint_as_float(s[g * 16]);
#pragma unroll
                    for (int c = 1; c < 16; ++c) y = fmaxf(y, __uint_as_float(s[g * 16 + c]));
                    if (y != -INFINITY) mx = fmaxf(mx, y * sc[g]);
                }
            }
            meet[b][half][i] = mx;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + wq) : "memory");
            mx = fmaxf(mx, meet[b][half ^ 1][i]);
            const bool moved = mx > m + kRefLazy || (m == -INFINITY && mx > -INFINITY);
            if (__any_sync(0xffffffffu, moved || top > ref)) {
                float al = 1.0f;
                if (moved) al = ex2(m - mx), m = mx, l *= al;
                if (top > ref) {
                    const uint32_t e = max(min((__float_as_uint(top) >> 23) + 1, 253u), 2u);     // 2^(e - 127) > top
                    al *= ref * __uint_as_float((254 - e) << 23);
                    ref = __uint_as_float(e << 23), per_ref = __uint_as_float((254 - e) << 23);
                }
                if (j > 0) {
                    wait(&pv_done[(j - 1) & 1], j - 1);
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = half * DH; c0 < half * DH + DH; c0 += 16) {
                        uint32_t o[16];
                        tm_ld16(mine + c0, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * al);
                        tm_st16(mine + c0, o);
                    }
                    tm_wait_st();
                }
            }
            if (j >= 2) wait(&pv_done[b], j - 2);                 // P's buffer is read
            const float z = m == -INFINITY ? 0.0f : kRefShift - m;
#pragma unroll 1
            for (int c0 = NH - 32; c0 >= 0; c0 -= 32) {
                uint32_t w[16], wl[LO ? 16 : 1];
                const int ca = half * NH + c0;
                if (c0 != NH - 32) tm_ld32(from + c0, s);
                const float sc[2] = {hd[0][ca / 16] * rf, hd[0][ca / 16 + 1] * rf};
                const float rv[2] = {hd[1][ca / 16] * per_ref, hd[1][ca / 16 + 1] * per_ref};
                if (c0 != NH - 32) {
                    tmem_wait_ld();
                    if (!all) see = seen(ca);
                }
                float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const int g = c / 16;
                    const float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), make_float2(sc[g], sc[g]), make_float2(z, z));
                    s[c] = __float_as_uint(ex2(x.x)), s[c + 1] = __float_as_uint(ex2(x.y));
                }
                if (!all) {
#pragma unroll
                    for (int c = 0; c < 32; ++c)
                        if (!(see >> c & 1)) s[c] = 0;
                }
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const int g = c / 16;
                    const float2 y = make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                    sum = __fadd2_rn(sum, y);
                    const float2 u = __fmul2_rn(y, make_float2(rv[g], rv[g]));
                    w[c / 2] = pack_f16(u.x, u.y);
                    if constexpr (LO) {
                        const float2 f = __half22float2(*(const __half2*) &w[c / 2]);
                        wl[c / 2] = pack_f16(u.x - f.x, u.y - f.y);
                    }
                }
                l += sum.x + sum.y;
                tm_st16(mine + P::kP + b * (N / 2) + ca / 2, w);
                if constexpr (LO) tm_st16(mine + P::kLow + b * (N / 2) + ca / 2, wl);
            }
            tm_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[b]), mbar_arrive(&p_full[b]);
        }
        if (n > 0) {
            wait(&pv_done[(n - 1) & 1], n - 1);
            tc_fence_after();
        }
        sums[half][i] = l;                                        // the row's sum from both halves
        asm volatile("bar.sync %0, 64;" ::"r"(1 + wq) : "memory");
        l += sums[half ^ 1][i];
        if (ok) {
            const float inv = l > 0.0f ? ref / l : l == l ? 0.0f : l;    // a row that sees no key is zero, a NaN row NaN
            const int64_t to = (int64_t) (q.tok + row / p.G) * p.o_tok + (int64_t) (h * p.G + row % p.G) * p.o_head;
#pragma unroll 1
            for (int c0 = half * DH; c0 < half * DH + DH; c0 += 32) {
                uint32_t o[32];
                if (n > 0) {
                    tm_ld32(mine + c0, o);
                    tmem_wait_ld();
                }
                if (row >= rows) continue;
#pragma unroll
                for (int c = 0; c < 32; c += 8) {
                    float x[8];
#pragma unroll
                    for (int u = 0; u < 8; ++u) x[u] = l != 0.0f ? __uint_as_float(o[c + u]) * inv : 0.0f;
                    store_row<8>(p.o, to + c0 + c, p.type, x, p.wide_out);
                }
            }
        }
    } else if (warp < kMmaWarp) {
        // ------------------------------------------------------------------------------------------------ codes
        // A thread converts chunk ct % CH of row ct / CH of every kRows tokens: 256 threads cover kRows / 16 groups of 16 tokens,
        // each within one block, so a chunk's address is its group's and a constant.
        constexpr int PER = N * CH / kConvThreads, kRows = kConvThreads / CH, GR = kRows / 16;
        const int ct = tid - 256, my_row = ct / CH, my_col = ct % CH, my_group = my_row / 16;
        const int32_t* tab = p.table + (int64_t) r * p.table_stride;
        const int shift = p.c.bs == 16 ? 4 : p.c.bs == 32 ? 5 : 6;
        // The table's entry of a token, as it is (tokens past the last that any row sees: the last one's); checked where it
        // is used, a tile later, so that nothing waits for it here.  Keys of a block outside the cache are read from block 0
        // and hidden by their header.
        auto entry = [&](int t) -> int { return __ldg(tab + (min(t, t_end - 1) >> shift)); };
        uint4 kr[PER], vr[PER];
        int ids[2][PER], head_id[2];                              // entries of this thread's groups, a tile ahead of their loads
        float hk = 0.0f, hv = 0.0f, hok = 0.0f;
        auto find = [&](int j, int s) {
#pragma unroll
            for (int i = 0; i < PER; ++i) ids[s][i] = entry(t_first + j * N + (i * GR + my_group) * 16);
            head_id[s] = entry(t_first + j * N + min(ct, NG - 1) * 16);
        };
        const int64_t mine = (int64_t) h * p.c.bs * D + (int64_t) (my_row % 16) * D + my_col * 16;
        const int8_t *k0 = p.c.k + mine, *v0 = p.c.v + mine;
        const uint32_t per_block = (uint32_t) (p.c.H * p.c.bs * D), in_block = (uint32_t) p.c.bs - 1;   // 65535 heads: below 2^31
        auto load = [&](int j, const int (&id)[PER], uint4 (&x)[PER], const int8_t* pool) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint32_t t = (uint32_t) (t_first + j * N + (i * GR + my_group) * 16);
                const uint32_t blk = (uint32_t) id[i] < (uint32_t) p.c.n_blocks ? (uint32_t) id[i] : 0u;
                x[i] = __ldg((const uint4*) (pool + ((uint64_t) blk * per_block + (t & in_block) * D)));
            }
        };
        auto load_head = [&](int j, int id) {
            if (ct < NG) {
                const bool ok = (uint32_t) id < (uint32_t) p.c.n_blocks && t_first + j * N + ct * 16 < t_end;
                const int64_t bh = (int64_t) (ok ? id : 0) * p.c.H + h;
                hk = __ldg(p.c.ks + bh), hv = __ldg(p.c.vs + bh), hok = ok ? 1.0f : 0.0f;
            }
        };
        const uint32_t to0 = (my_col >> 2) * (N * 128) + sw128(my_row, (my_col & 3) * 2), to1 = (my_col >> 2) * (N * 128) + sw128(my_row, (my_col & 3) * 2 + 1);
        auto store = [&](const uint4 (&x)[PER], uint8_t* to) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                uint4 a, d;
                codes4(x[i].x, a.x, a.y), codes4(x[i].y, a.z, a.w), codes4(x[i].z, d.x, d.y), codes4(x[i].w, d.z, d.w);
                *(uint4*) (to + to0 + i * (kRows * 128)) = a;
                *(uint4*) (to + to1 + i * (kRows * 128)) = d;
            }
            fence_proxy_async();
            __syncwarp();
        };
        if (n > 0) {
            find(0, 0);
            load(0, ids[0], kr, k0), load_head(0, head_id[0]), load(0, ids[0], vr, v0);
            find(1, 1);
        }
        auto step = [&](int j, auto odd) -> bool {                // ids[1 - odd] are tile j + 1's, ids[odd] free for j + 2's
            constexpr int b = decltype(odd)::value;
            bool go = true;
            if (j >= 2) go = mbar_wait_bounded(&k_empty[b], ((j - 2) >> 1) & 1, p.err, kSitePrompt);
            if (!__all_sync(0xffffffffu, go)) return false;
            if (ct < NG) heads[j & 3][0][ct] = hok != 0.0f ? hk : 0.0f, heads[j & 3][1][ct] = hok != 0.0f ? hv : 0.0f, heads[j & 3][2][ct] = hok;
            store(kr, ks + b * P::kKV);
            if (lane == 0) mbar_arrive(&k_full[b]);
            if (j + 1 < n) load(j + 1, ids[1 - b], kr, k0), load_head(j + 1, head_id[1 - b]);
            find(j + 2, b);
            if (j >= 2) go = mbar_wait_bounded(&v_empty[b], ((j - 2) >> 1) & 1, p.err, kSitePrompt);
            if (!__all_sync(0xffffffffu, go)) return false;
            store(vr, vs + b * P::kKV);
            if (lane == 0) mbar_arrive(&v_full[b]);
            if (j + 1 < n) load(j + 1, ids[1 - b], vr, v0);
            return true;
        };
        for (int j = 0; j < n; j += 2) {
            if (!step(j, std::integral_constant<int, 0>{})) break;
            if (j + 1 < n && !step(j + 1, std::integral_constant<int, 1>{})) break;
        }
    } else {
        // ------------------------------------------------------------------------------------------------ products
        constexpr uint32_t qk = (1u << 4) | ((uint32_t) (N >> 3) << 17) | (8u << 24);
        constexpr uint32_t pv = (1u << 4) | (1u << 16) | ((uint32_t) (D >> 3) << 17) | (8u << 24);
        const uint64_t qd = pf_sdesc(smem_u32(qs)), kd = pf_sdesc(smem_u32(ks)), vd = mn_desc(smem_u32(vs), N * 128);
        auto waits = [&](uint64_t* bar, int j) -> bool {
            return __all_sync(0xffffffffu, mbar_wait_bounded(bar, (j >> 1) & 1, p.err, kSitePrompt));
        };
        auto scores = [&](int j) -> bool {
            const int b = j & 1;
            if (!waits(&k_full[b], j)) return false;
            if (j >= 2 && !waits(&s_free[b], j - 2)) return false;
            tc_fence_after();
            const uint64_t kb = kd + (uint32_t) (b * (P::kKV >> 4));
            const uint32_t to = tmem + P::kS + b * N;
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                umma_ss(to, qd + (((k >> 2) * 16384 + (k & 3) * 32) >> 4), kb + (((k >> 2) * (N * 128) + (k & 3) * 32) >> 4), qk, k > 0);
            if (lane == 0) mbar_arrive(&s_full[b]);               // hands the converters' scales on
            umma_commit(&s_full[b]);
            umma_commit(&k_empty[b]);
            return true;
        };
        bool ok = n > 0 && scores(0);
        for (int j = 0; j < n && ok; ++j) {
            const int b = j & 1;
            if (j + 1 < n && !(ok = scores(j + 1))) break;
            ok = waits(&p_full[b], j) && waits(&v_full[b], j);
            if (!ok) break;
            tc_fence_after();
            const uint64_t vb = vd + (uint32_t) (b * (P::kKV >> 4));
            const uint32_t from = tmem + P::kP + b * (N / 2);
#pragma unroll
            for (int k = 0; k < N / 16; ++k) umma_ts(tmem, from + k * 8, vb + ((k * 2048) >> 4), pv, (j | k) != 0);
            if constexpr (LO) {
#pragma unroll
                for (int k = 0; k < N / 16; ++k) umma_ts(tmem, from + (P::kLow - P::kP) + k * 8, vb + ((k * 2048) >> 4), pv, 1);
            }
            umma_commit(&v_empty[b]);
            umma_commit(&pv_done[b]);
        }
        if (!ok && n > 0) {                                       // every product so far, the scores ahead among them
            umma_commit(&drained);
            mbar_drain(&drained, 0, p.err, kSitePrompt);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

}  // namespace
}  // namespace tsb
