// tsb_cache_prompt.cuh - attention of many queries over the 8-bit cache on tcgen05 (16-bit queries): part of tsb_cache.cu.
//
// CTA (tile of 128 rows, key / value head, request); rows are query tokens times the heads of the group, so a grouped model
// reads a key for all of them.  Keys and values in tiles of kN tokens, two stages each:
//   warps 0-3   softmax: a thread a row (a tensor-memory lane); scores from tensor memory, weights back to it as fp16
//   warps 4-11  the codes from the cache to fp16 operands in shared memory (exact: the product needs 16-bit operands, and
//               int8 products would take three planes of the queries and three tensor-memory reads a score)
//   warp 12     one thread issues the products: S = Q K^T (both K-major), O += P V (P in tensor memory, V as it lies, its
//               value columns contiguous: MN-major)
// S and P are double buffered, so the products of tile j + 1 and j - 1 run while tile j is in the softmax.  O stays in tensor
// memory; its rows are rescaled only when a row's score exceeds its reference by 2^4 (or a block's value scale the
// largest so far), which after a row's first tiles is rare.
// Weights are exp2(x - reference + 11), at most 2^15, times the block's value scale relative to the largest so far: fp16 keeps
// 11 bits of those down to 2^-25 of the reference.  The sums l and everything of the softmax are fp32.
// What bounds it: at head_dim 256 the products (4 * 128 * 64 * 256 a tile), at 64 the exponentials.
#pragma once

#include "tsb_tc.cuh"

namespace tsb {
namespace {

constexpr unsigned kSitePrompt = 0xC0000001u;   // the error word when a wait of this kernel gave up
constexpr int kPromptThreads = 13 * 32, kConvThreads = 8 * 32;
constexpr float kRefShift = 11.0f, kRefLazy = 4.0f;

template <int D>
struct Prompt {
    static constexpr int kN = D == 256 ? 64 : 128;
    static constexpr int kQ = 128 * D * 2, kKV = kN * D * 2;
    static constexpr int kGroups = kN / 16;
    // tensor memory columns: O, S twice, P twice (two weights a column)
    static constexpr int kS = D, kP = D + 2 * kN;
    static_assert(kP + kN <= 512, "tensor memory");
    static constexpr int kSmem = kQ + 4 * kKV + 1024;                      // and room to align
    static constexpr int kAsk = kSmem > 120 * 1024 ? kSmem : 120 * 1024;   // one CTA a SM: each takes all of tensor memory
};
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr, int chunk_bytes) {   // MN-major, 128-byte swizzle
    return (uint64_t) ((addr >> 4) & 0x3FFFu) | ((uint64_t) (chunk_bytes >> 4) << 16) | ((uint64_t) (1024 >> 4) << 32) |
           ((uint64_t) 1 << 46) | ((uint64_t) 2 << 61);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"(acc)
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
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::TSB_W8(r, 0),
                 TSB_W8(r, 8), TSB_W8(r, 16), TSB_W8(r, 24), "r"(addr)
                 : "memory");
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

template <int D>
__global__ void __launch_bounds__(kPromptThreads, 1) k_attn_prompt(const __grid_constant__ AttnParams p) {
    using P = Prompt<D>;
    constexpr int N = P::kN, NG = P::kGroups, CH = D / 16;       // CH: 16-code chunks of a token
    extern __shared__ __align__(1024) uint8_t prompt_smem[];
    uint8_t* smem = prompt_smem + ((1024 - (smem_u32(prompt_smem) & 1023)) & 1023);
    __shared__ uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], s_free[2], p_full[2], pv_done[2];
    __shared__ uint32_t tbase;
    __shared__ float rowf[128];
    __shared__ float heads[4][3][NG];                             // key scales, value scales, whether the block is in the cache
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rt = gridDim.x - 1 - blockIdx.x, h = blockIdx.y, r = blockIdx.z;
    const Req q = attn_req(p, r);
    const int rows = q.n * p.G;
    if (rt * 128 >= rows) return;
    int first, steps;
    tile_steps<128>(p, q, rt, first, steps);
    const int t_first = first * kStep, t_end = (first + steps) * kStep, n = (steps * kStep + N - 1) / N;
    uint8_t *qs = smem, *ks = smem + P::kQ, *vs = ks + 2 * P::kKV;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 8), mbar_init(&k_empty[i], 1), mbar_init(&v_full[i], 8), mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 2), mbar_init(&s_free[i], 4), mbar_init(&p_full[i], 4), mbar_init(&pv_done[i], 1);
        }
        fence_mbar_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tbase)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // the rows, scaled by a power of two to [2^10, 2^11) at their largest: exact in fp16 down to 2^-35 of it
    for (int i = warp; i < 128; i += 13) {
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

    if (warp < 4) {
        // ------------------------------------------------------------------------------------------------ softmax
        const uint32_t mine = tmem + ((uint32_t) (warp * 32) << 16);
        const int i = warp * 32 + lane, row = rt * 128 + i;
        const int pos = q.len - q.n + min(row, rows - 1) / p.G;
        const int pmin = q.len - q.n + (rt * 128) / p.G;
        const int lmax = p.window > 0 ? q.len - q.n + (min(rt * 128 + 128, rows) - 1) / p.G - p.window + 1 : INT_MIN;
        const int win = p.window > 0 ? p.window : INT_MAX;
        const float rf = rowf[i];
        float m = -INFINITY, l = 0.0f, ref = 0.0f, per_ref = 0.0f;
        bool ok = true;
        for (int j = 0; j < n && ok; ++j) {
            const int b = j & 1, t0 = t_first + j * N;
            ok = mbar_wait_bounded(&s_full[b], (j >> 1) & 1, p.err, kSitePrompt);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const float(*hd)[NG] = heads[j & 3];
            const bool edge = t0 + N - 1 > pmin || t0 < lmax || t0 + N > t_end;
            auto hidden = [&](int c) {                            // column c of the tile
                const int t = t0 + c;
                return t > pos || pos - t >= win || hd[2][c >> 4] == 0.0f;
            };
            // a group outside the cache hides its keys; inside a tile that cuts nothing else this is rare
            bool holes = edge;
            float top = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) holes |= hd[2][g] == 0.0f, top = fmaxf(top, hd[1][g]);
            float mx = -INFINITY;
#pragma unroll
            for (int c0 = 0; c0 < N; c0 += 32) {
                uint32_t s[32];
                tm_ld32(mine + P::kS + b * N + c0, s);
                tmem_wait_ld();
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    float y = -INFINITY;
                    if (holes) {
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            if (!hidden(c0 + g * 16 + c)) y = fmaxf(y, __uint_as_float(s[g * 16 + c]));
                    } else {
#pragma unroll
                        for (int c = 0; c < 16; ++c) y = fmaxf(y, __uint_as_float(s[g * 16 + c]));
                    }
                    if (y != -INFINITY) mx = fmaxf(mx, y * (hd[0][c0 / 16 + g] * rf));
                }
            }
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
                    ok = mbar_wait_bounded(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1, p.err, kSitePrompt);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < D; c0 += 32) {
                        uint32_t o[32];
                        tm_ld32(mine + c0, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * al);
                        tm_st32(mine + c0, o);
                    }
                    tm_wait_st();
                }
            }
            if (j >= 2) {                                         // P's buffer is read
                ok = mbar_wait_bounded(&pv_done[b], ((j - 2) >> 1) & 1, p.err, kSitePrompt);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
            }
            const float z = m == -INFINITY ? 0.0f : kRefShift - m;
#pragma unroll
            for (int c0 = 0; c0 < N; c0 += 32) {
                uint32_t s[32], w[16];
                tm_ld32(mine + P::kS + b * N + c0, s);
                tmem_wait_ld();
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const float sc = hd[0][c0 / 16 + g] * rf, rv = hd[1][c0 / 16 + g] * per_ref;
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        float a = ex2(fmaf(__uint_as_float(s[g * 16 + c]), sc, z)), d = ex2(fmaf(__uint_as_float(s[g * 16 + c + 1]), sc, z));
                        if (holes) {
                            if (hidden(c0 + g * 16 + c)) a = 0.0f;
                            if (hidden(c0 + g * 16 + c + 1)) d = 0.0f;
                        }
                        l += a + d;
                        w[g * 8 + c / 2] = pack_f16(a * rv, d * rv);
                    }
                }
                tm_st16(mine + P::kP + b * (N / 2) + c0 / 2, w);
            }
            tm_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[b]), mbar_arrive(&p_full[b]);
        }
        if (ok && n > 0) {
            ok = mbar_wait_bounded(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1, p.err, kSitePrompt);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
        }
        if (ok) {
            const float inv = l > 0.0f ? ref / l : l == l ? 0.0f : l;    // a row that sees no key is zero, a NaN row NaN
            const int64_t to = (int64_t) (q.tok + row / p.G) * p.o_tok + (int64_t) (h * p.G + row % p.G) * p.o_head;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
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
    } else if (warp < 12) {
        // ------------------------------------------------------------------------------------------------ codes
        constexpr int PER = N * CH / kConvThreads;               // chunks a thread of a tile
        const int ct = tid - 128;
        const int32_t* tab = p.table + (int64_t) r * p.table_stride;
        const int shift = p.c.bs == 16 ? 4 : p.c.bs == 32 ? 5 : 6;
        auto block_of = [&](int t) -> int {                       // -1: past the keys that any row sees, or outside the cache
            if (t >= t_end) return -1;
            const int id = __ldg(tab + (t >> shift));
            return id < p.c.n_blocks ? max(id, -1) : -1;
        };
        uint4 kr[PER], vr[PER];
        float hk = 0.0f, hv = 0.0f, hok = 0.0f;
        auto load = [&](int j, uint4 (&x)[PER], const int8_t* pool) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int c = i * kConvThreads + ct, t = t_first + j * N + c / CH;
                const int id = block_of(t);
                x[i] = make_uint4(0, 0, 0, 0);
                if (id >= 0) x[i] = *(const uint4*) (pool + (((int64_t) id * p.c.H + h) * p.c.bs + (t & (p.c.bs - 1))) * D + (c % CH) * 16);
            }
        };
        auto load_head = [&](int j) {
            if (ct < NG) {
                const int id = block_of(t_first + j * N + ct * 16);
                const int64_t bh = (int64_t) max(id, 0) * p.c.H + h;
                hk = id >= 0 ? p.c.ks[bh] : 0.0f, hv = id >= 0 ? p.c.vs[bh] : 0.0f, hok = id >= 0 ? 1.0f : 0.0f;
            }
        };
        auto store = [&](const uint4 (&x)[PER], uint8_t* to) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int c = i * kConvThreads + ct, t = c / CH, cc = c % CH;
                uint4 a, d;
                codes4(x[i].x, a.x, a.y), codes4(x[i].y, a.z, a.w), codes4(x[i].z, d.x, d.y), codes4(x[i].w, d.z, d.w);
                uint8_t* tile = to + (cc >> 2) * (N * 128);
                *(uint4*) (tile + sw128(t, (cc & 3) * 2)) = a;
                *(uint4*) (tile + sw128(t, (cc & 3) * 2 + 1)) = d;
            }
            fence_proxy_async();
            __syncwarp();
        };
        bool ok = true;
        if (n > 0) load(0, kr, p.c.k), load_head(0), load(0, vr, p.c.v);
        for (int j = 0; j < n && ok; ++j) {
            const int b = j & 1;
            if (j >= 2) ok = mbar_wait_bounded(&k_empty[b], ((j - 2) >> 1) & 1, p.err, kSitePrompt);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (ct < NG) heads[j & 3][0][ct] = hk, heads[j & 3][1][ct] = hv, heads[j & 3][2][ct] = hok;
            store(kr, ks + b * P::kKV);
            if (lane == 0) mbar_arrive(&k_full[b]);
            if (j + 1 < n) load(j + 1, kr, p.c.k), load_head(j + 1);
            if (j >= 2) ok = mbar_wait_bounded(&v_empty[b], ((j - 2) >> 1) & 1, p.err, kSitePrompt);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            store(vr, vs + b * P::kKV);
            if (lane == 0) mbar_arrive(&v_full[b]);
            if (j + 1 < n) load(j + 1, vr, p.c.v);
        }
    } else if (lane == 0) {
        // ------------------------------------------------------------------------------------------------ products
        constexpr uint32_t qk = (1u << 4) | ((uint32_t) (N >> 3) << 17) | (8u << 24);
        constexpr uint32_t pv = (1u << 4) | (1u << 16) | ((uint32_t) (D >> 3) << 17) | (8u << 24);
        const uint32_t qa = smem_u32(qs), ka = smem_u32(ks), va = smem_u32(vs);
        bool ok = true;
        auto scores = [&](int j) -> bool {
            const int b = j & 1;
            if (!mbar_wait_bounded(&k_full[b], (j >> 1) & 1, p.err, kSitePrompt)) return false;
            if (j >= 2 && !mbar_wait_bounded(&s_free[b], ((j - 2) >> 1) & 1, p.err, kSitePrompt)) return false;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
                umma_ss(tmem + P::kS + b * N, pf_sdesc(qa + (k >> 2) * 16384 + (k & 3) * 32), pf_sdesc(ka + b * P::kKV + (k >> 2) * (N * 128) + (k & 3) * 32),
                        qk, k > 0);
            mbar_arrive(&s_full[b]);                              // hands the converters' scales on
            pf_commit(&s_full[b]);
            pf_commit(&k_empty[b]);
            return true;
        };
        if (n > 0) ok = scores(0);
        int done = 0;
        for (int j = 0; j < n && ok; ++j) {
            const int b = j & 1;
            if (j + 1 < n && !(ok = scores(j + 1))) break;
            ok = mbar_wait_bounded(&p_full[b], (j >> 1) & 1, p.err, kSitePrompt) && mbar_wait_bounded(&v_full[b], (j >> 1) & 1, p.err, kSitePrompt);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int k = 0; k < N / 16; ++k)
                umma_ts(tmem, tmem + P::kP + b * (N / 2) + k * 8, mn_desc(va + b * P::kKV + k * 2048, N * 128), pv, j > 0 || k > 0);
            pf_commit(&v_empty[b]);
            pf_commit(&pv_done[b]);
            ++done;
        }
        // products in flight end before the CTA's memory goes
        if (!ok && done > 0) mbar_wait_bounded(&pv_done[(done - 1) & 1], ((done - 1) >> 1) & 1, p.err, kSitePrompt);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

}  // namespace
}  // namespace tsb
