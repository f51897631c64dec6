// tsb_cache.cu - the paged 8-bit key / value cache of a serving step: block tables and slot maps from the requests'
// lengths, appending and reading back tokens, and attention over the cache.
//
// The cache is two pools of int8 codes [n_blocks][n_kv_heads][block_size][head_dim] with one fp32 scale per (block, head):
// a key or value is code * scale.  The tokens of one (block, head) are contiguous, so a warp that attends 16 tokens
// reads 16 * head_dim consecutive bytes, and every token of such a step shares one scale.
#include "../../include/tsb_moe.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "tsb_device.cuh"
#include "tsb_warp_mma.cuh"

namespace tsb {

void set_last_error(const char* msg);   // tsb_moe.cu: the text tsb_last_error returns

namespace {

int cfail(int code, const char* fmt, ...) {
    char b[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(b, sizeof b, fmt, ap);
    va_end(ap);
    set_last_error(b);
    return code;
}
int ccuda(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cfail(TSB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    return TSB_OK;
}
cudaStream_t cst(void* s) { return (cudaStream_t) s; }

int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return n;
}

// ------------------------------------------------------------------------------------------------ block tables
constexpr int kTabThreads = 512;
constexpr int kTabMaxReq = 8192;

struct TabParams {
    const int32_t *lens, *n_new;
    const uint8_t* done;
    int n_req;
    int32_t* table;
    int64_t table_stride;
    int width;
    int32_t* free_list;
    int cap_free;
    const int32_t* n_free;
    int block_size;
    int32_t *lens_out, *cu_new;
    int64_t* slots;
    int64_t cap_tokens;
    int32_t* n_free_out;
};

// What request r brings: its cached tokens, the tokens it adds, the blocks it gives back and those it takes (0 when
// they would not fit its table row).
struct TabReq {
    int len, add, gives, has, takes;
    bool fits, done;
};
__device__ __forceinline__ TabReq tab_req(const TabParams& p, int r) {
    TabReq q;
    q.len = max(p.lens[r], 0);
    q.add = max(p.n_new[r], 0);
    q.done = p.done && p.done[r] != 0;
    q.has = (int) (((int64_t) q.len + p.block_size - 1) / p.block_size);
    const int64_t after = ((int64_t) q.len + q.add + p.block_size - 1) / p.block_size;
    q.fits = !q.done && after <= p.width;
    q.gives = q.done ? min(q.has, p.width) : 0;
    q.takes = q.fits ? (int) (after - q.has) : 0;
    return q;
}

// The largest i in [0, n] with a[i] <= v (a ascending, a[0] <= v).
__device__ __forceinline__ int last_le(const int* a, int n, int64_t v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((int64_t) a[mid] <= v) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// One launch.  Every CTA scans the requests itself (three prefix sums in shared memory: tokens added, blocks taken,
// blocks given back; a few thousand requests are a few words a thread), then all CTAs share the blocks and the tokens:
// which block a token's position lands in follows from the prefix sums alone, so no CTA reads what another writes.
// The stack of free blocks is free_list[0 .. n_free) with the blocks given back on top of it; the k-th block taken is
// the k-th from the top.  What bounds it is the launch and the dependent loads (lengths, then list or table): at 8
// requests nothing else is left, at 1000 requests and 33,000 tokens the slots' 8 bytes a token are 0.3 MB.
__global__ void __launch_bounds__(kTabThreads) k_block_tables(const TabParams p) {
    extern __shared__ int sh[];
    const int R = p.n_req;
    int* cu = sh;                     // R + 1
    int* take = sh + (R + 1);         // R + 1
    int* give = sh + 2 * (R + 1);     // R + 1
    __shared__ int wsum[3][kTabThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (R + kTabThreads - 1) / kTabThreads;
    const int r0 = min(tid * per, R), r1 = min(r0 + per, R);
    int s[3] = {0, 0, 0};
    for (int r = r0; r < r1; ++r) {
        const TabReq q = tab_req(p, r);
        s[0] += q.add, s[1] += q.takes, s[2] += q.gives;
    }
    int x[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        int v = s[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) wsum[i][warp] = v;
        x[i] = v - s[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        for (int w = 0; w < warp; ++w) x[i] += wsum[i][w];
    }
    for (int r = r0; r < r1; ++r) {
        const TabReq q = tab_req(p, r);
        cu[r] = x[0], take[r] = x[1], give[r] = x[2];
        x[0] += q.add, x[1] += q.takes, x[2] += q.gives;
    }
    if (tid == kTabThreads - 1) cu[R] = x[0], take[R] = x[1], give[R] = x[2];
    __syncthreads();

    const int held = min(max(*p.n_free, 0), p.cap_free);
    const int given = min(give[R], p.cap_free - held);
    const int have = held + given;
    const int granted = take[last_le(take, R, have)];     // requests are served in order while their blocks last
    auto stack = [&](int i) -> int {                      // the i-th block from the bottom
        if (i < held) return p.free_list[i];
        const int r = last_le(give, R, i - held);
        return p.table[(int64_t) r * p.table_stride + (i - held - give[r])];
    };
    const int64_t g = (int64_t) blockIdx.x * kTabThreads + tid, step = (int64_t) gridDim.x * kTabThreads;
    for (int64_t r = g; r < R; r += step) {
        const TabReq q = tab_req(p, (int) r);
        const bool ok = q.fits && (q.takes == 0 || take[r + 1] <= have);
        p.lens_out[r] = q.done ? 0 : ok ? q.len + q.add : q.len;
        p.cu_new[r] = cu[r];
    }
    if (g == 0) {
        p.cu_new[R] = cu[R];
        *p.n_free_out = have - granted;
    }
    for (int64_t i = g; i < given; i += step) p.free_list[held + i] = stack(held + (int) i);
    for (int64_t k = g; k < granted; k += step) {
        const int r = last_le(take, R, k);
        const TabReq q = tab_req(p, r);
        p.table[(int64_t) r * p.table_stride + q.has + (k - take[r])] = stack(have - 1 - (int) k);
    }
    for (int64_t t = g; t < p.cap_tokens; t += step) {
        int64_t slot = -1;
        if (t < cu[R]) {
            const int r = last_le(cu, R, t);
            const TabReq q = tab_req(p, r);
            if (q.fits && (q.takes == 0 || take[r + 1] <= have)) {
                const int64_t pos = (int64_t) q.len + (t - cu[r]);
                const int j = (int) (pos / p.block_size);
                const int b = j < q.has ? p.table[(int64_t) r * p.table_stride + j]
                                        : stack(have - 1 - (take[r] + (j - q.has)));
                slot = b < 0 ? -1 : (int64_t) b * p.block_size + pos % p.block_size;
            }
        }
        p.slots[t] = slot;
    }
}

// ------------------------------------------------------------------------------------------------ append, read back
struct Cache {
    int8_t *k, *v;
    float *ks, *vs;
    int n_blocks, bs, H, D;
};

struct AppendParams {
    Cache c;
    const void *k, *v;
    int type;
    int64_t k_tok, k_head, v_tok, v_head;
    const int64_t* slots;
    int64_t n_tok;
    int per_cta;      // tokens whose runs a CTA starts
    bool wide;
};

constexpr float kCodeMax = 127.0f;
// A value as it enters the cache: NaN counts as 0 and an infinity as the largest finite value, so that one bad element
// cannot make a whole block's codes undefined.
__device__ __forceinline__ float cache_value(float x) {
    if (x != x) return 0.0f;
    return fminf(fmaxf(x, -3.3895314e38f), 3.3895314e38f);   // the largest finite bf16
}
__device__ __forceinline__ int cache_code(float x, float scale) {
    return scale > 0.0f ? (int) fminf(fmaxf(rintf(x / scale), -kCodeMax), kCodeMax) : 0;
}

// CTA (chunk of per_cta tokens, head).  A run is the tokens of one call that follow one another within one cache block;
// its first token is the leader, and one warp takes a run's keys or values: the largest magnitude over the run, the
// block's new scale max(old, largest / 127) (old: none when the run starts the block), the block's earlier codes
// brought to it when it grew, and the run's codes.  One warp owns the (block, head), so no value is written twice and
// nothing is atomic.  Divisions are IEEE: the same codes on any device.  Bound by the rows' bytes: the second pass over
// a run reads it from L1.
__global__ void __launch_bounds__(256) k_kv8_append(const AppendParams p) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int h = blockIdx.y;
    const int bs = p.c.bs, D = p.c.D, DV = D / 8;
    const int64_t t0 = (int64_t) blockIdx.x * p.per_cta, cap = (int64_t) p.c.n_blocks * bs;
    const int64_t mine = t0 + lane;
    bool leads = false;
    if (lane < p.per_cta && mine < p.n_tok) {
        const int64_t s = p.slots[mine];
        if (s >= 0 && s < cap) leads = mine == 0 || s % bs == 0 || p.slots[mine - 1] != s - 1;
    }
    unsigned todo = __ballot_sync(0xffffffffu, leads);
    for (int job = 0; todo; ++job) {
        const int at = __ffs(todo) - 1;
        if (job & 1) todo &= todo - 1;
        if ((job & 7) != warp) continue;
        const bool is_v = job & 1;
        const int64_t t = t0 + at, s = p.slots[t], blk = s / bs;
        const int off = (int) (s - blk * bs);
        int n = 0;                                       // tokens of the run
        for (int base = 0; base < bs - off; base += 32) {
            const int i = base + lane;
            const bool in = i < bs - off && t + i < p.n_tok && p.slots[t + i] == s + i;
            const unsigned b = __ballot_sync(0xffffffffu, in);
            n += b == 0xffffffffu ? 32 : __ffs(~b) - 1;
            if (b != 0xffffffffu) break;
        }
        const void* src = is_v ? p.v : p.k;
        const int64_t row = is_v ? p.v_tok : p.k_tok, col = (is_v ? p.v_head : p.k_head) * h;
        int8_t* codes = (is_v ? p.c.v : p.c.k) + (blk * p.c.H + h) * (int64_t) bs * D;
        float* sp = (is_v ? p.c.vs : p.c.ks) + blk * p.c.H + h;
        float peak = 0.0f;
        for (int e = lane; e < n * DV; e += 32) {
            float x[8];
            load8(x, src, (t + e / DV) * row + col + (e % DV) * 8, p.type, p.wide);
#pragma unroll
            for (int j = 0; j < 8; ++j) peak = fmaxf(peak, fabsf(cache_value(x[j])));
        }
        peak = warp_max(peak);
        const float was = off > 0 ? *sp : 0.0f;
        const float now = fmaxf(was, peak / kCodeMax);
        __syncwarp();
        if (lane == 0) *sp = now;
        if (off > 0 && now != was) {
            const float ratio = was / now;
            for (int e = lane; e < off * D / 16; e += 32) {
                uint4 w = ((const uint4*) codes)[e];
                uint32_t* u = (uint32_t*) &w;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t r = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        r |= (uint32_t) (uint8_t) (int8_t) rintf((float) (int8_t) (u[i] >> (8 * j)) * ratio) << (8 * j);
                    u[i] = r;
                }
                ((uint4*) codes)[e] = w;
            }
        }
        for (int e = lane; e < n * DV; e += 32) {
            float x[8];
            load8(x, src, (t + e / DV) * row + col + (e % DV) * 8, p.type, p.wide);
            uint32_t u[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) u[j >> 2] |= (uint32_t) (uint8_t) cache_code(cache_value(x[j]), now) << (8 * (j & 3));
            *(uint2*) (codes + (int64_t) off * D + (int64_t) e * 8) = make_uint2(u[0], u[1]);
        }
    }
}

// One thread per 16 values of a (token, head): key and value.  A slot outside the cache reads as zeros.
__global__ void __launch_bounds__(256) k_kv8_read(const Cache c, const int64_t* __restrict__ slots, int64_t n_tok,
                                                  void* k, void* v, int type) {
    const int per = c.D / 16;
    const int64_t e = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (e >= n_tok * c.H * per) return;
    const int64_t th = e / per, t = th / c.H;
    const int h = (int) (th - t * c.H), part = (int) (e - th * per);
    const int64_t s = slots[t];
    const bool ok = s >= 0 && s < (int64_t) c.n_blocks * c.bs;
    const int64_t blk = ok ? s / c.bs : 0, bh = blk * c.H + h;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const int8_t* codes = (w ? c.v : c.k) + (bh * c.bs + (ok ? s - blk * c.bs : 0)) * c.D + part * 16;
        const uint4 q = ok ? *(const uint4*) codes : make_uint4(0, 0, 0, 0);
        const float sc = ok ? (w ? c.vs : c.ks)[bh] : 0.0f;
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
        float f[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) f[j] = (float) (int8_t) (u[j >> 2] >> (8 * (j & 3))) * sc;
        void* out = w ? v : k;
        if (type == E_F32) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                ((float4*) out)[e * 4 + j] = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
        } else {
            uint32_t r[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                r[j] = type == E_F16 ? pack_f16(f[2 * j], f[2 * j + 1]) : pack_bf16(f[2 * j], f[2 * j + 1]);
            ((uint4*) out)[e * 2] = make_uint4(r[0], r[1], r[2], r[3]);
            ((uint4*) out)[e * 2 + 1] = make_uint4(r[4], r[5], r[6], r[7]);
        }
    }
}

// ------------------------------------------------------------------------------------------------ attention
constexpr int kAttnWarps = 4;
constexpr int kStep = 16;            // tokens of a step: one matrix-product depth, always within one cache block
constexpr int kSplitRows = 64;       // rows a key / value head has (queries x heads of its group) up to which the
                                     // steps of a request are split over CTAs
constexpr int kMaxReq = 4096;

struct AttnParams {
    Cache c;
    const void* q;
    void* o;
    int type, n_req, G, max_q, window;
    float scale_log2;                // scale * log2(e)
    int64_t q_tok, q_head, o_tok, o_head, n_tok;
    const int32_t* table;
    int64_t table_stride;
    int width;
    const int32_t *lens, *cu;
    int tiles;                       // 16-row tiles of the longest request
    // split over CTAs: steps before each request, partial rows
    int64_t* pre;                    // [n_req + 1]
    float* part;                     // [2 * CTAs][16][D], then their maxima and sums [2 * CTAs][2][16]
    int n_cta;
};

struct Req {
    int len, n, tok;                 // cached tokens, queries, first query's row in q
};
__device__ __forceinline__ Req attn_req(const AttnParams& p, int r) {
    Req q;
    q.len = (int) min((int64_t) max(p.lens[r], 0), (int64_t) p.width * p.c.bs);
    if (p.cu) {
        q.tok = max(p.cu[r], 0);
        q.n = min(p.cu[r + 1] - q.tok, p.max_q);
        q.n = (int) max((int64_t) 0, min((int64_t) q.n, p.n_tok - q.tok));
    } else {
        q.tok = r * p.max_q;
        q.n = p.max_q;
    }
    return q;
}
// The steps [first, first + n) that the rows of tile rt see.
__device__ __forceinline__ void tile_steps(const AttnParams& p, const Req& q, int rt, int& first, int& n) {
    const int rows = q.n * p.G, r0 = rt * 16;
    first = n = 0;
    if (r0 >= rows) return;
    const int i0 = r0 / p.G, i1 = (min(r0 + 16, rows) - 1) / p.G;
    const int hi = q.len - q.n + i1 + 1, lo = p.window > 0 ? max(0, q.len - q.n + i0 - p.window + 1) : 0;
    if (hi <= 0) return;
    first = lo / kStep;
    n = (hi + kStep - 1) / kStep - first;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint4 ld_code16(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ld_code8(const int8_t* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
// Four codes (bytes biased by 128) as fp16 values, exactly: byte b under the high byte 0x64 is the fp16 number 1024 + b.
__device__ __forceinline__ uint32_t half_pair(uint32_t biased, uint32_t sel) {
    const uint32_t w = __byte_perm(biased, 0x64646464u, sel);
    const __half2 r = __hsub2(*(const __half2*) &w, __floats2half2_rn(1152.0f, 1152.0f));
    return *(const uint32_t*) &r;
}

// The rows of one tile as left operands, in shared memory [SP][D / 16][32 lanes]: row values in fp16 after a power-of-two
// scale that brings the row's largest magnitude to [1024, 2048) (rowf undoes it), as one fp16 value (SP 1: exact for
// 16-bit inputs down to 2^-25 of the row's largest) or as two (SP 2, 22 bits, for fp32 inputs).  The order of the
// contraction is the order in which a lane reads codes: 16 consecutive bytes are four depths of 16.
template <int D, int SP>
__device__ __forceinline__ void stage_rows(const AttnParams& p, const Req& q, int h, int rt, uint4* qf, float* rowf,
                                           int warp, int n_warps, int lane) {
    const int rows = q.n * p.G;
    for (int i = warp; i < 16; i += n_warps) {
        const int row = rt * 16 + i;
        float x[D / 32];
        float peak = 0.0f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            x[j] = row < rows ? load_elem(p.q, (int64_t) (q.tok + row / p.G) * p.q_tok + (int64_t) (h * p.G + row % p.G) * p.q_head +
                                                   j * 32 + lane,
                                          p.type)
                              : 0.0f;
            peak = fmaxf(peak, fabsf(x[j]));
        }
        peak = warp_max(peak);
        const int e = (int) ((__float_as_uint(peak) >> 23) & 255u);              // 2^(e - 127) <= peak
        const int up = e == 0 || e == 255 ? 0 : min(max(137 - e, -126), 126);    // to [1024, 2048)
        const float f = __uint_as_float((uint32_t) (127 + up) << 23);
        if (lane == 0) rowf[i] = p.scale_log2 * __uint_as_float((uint32_t) (127 - up) << 23);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
            // value d of row i: chunk d / 64, quad (d / 16) % 4, byte d % 16 -> depth byte / 4, register and half
            const int d = j * 32 + lane, b = d & 15;
            const int slot = ((d >> 6) * 4 + (b >> 2)) * 32 + (i & 7) * 4 + ((d >> 4) & 3);
            const int at = ((b & 2) ? 4 : 0) + ((i & 8) ? 2 : 0) + (b & 1);      // half index in {a0, a1, a2, a3}
            const float y = x[j] * f;
            const __half hi = __float2half_rn(y);
            ((__half*) (qf + slot))[at] = hi;
            if (SP == 2) ((__half*) (qf + (D / 16) * 32 + slot))[at] = __float2half_rn(y - __half2float(hi));
        }
    }
}

// A warp's running rows: row g = lane / 4 and row g + 8 of the tile, output columns as the lane's value bytes.
template <int D>
struct Rows {
    float o[D / 8][4];
    float m[2], l[2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.0f;
    }
};

template <int D>
struct Codes {
    static constexpr int KC = D / 64, VC = D / 128 > 0 ? D / 128 : 1;
    uint4 k[2][KC], v[4][VC];
    float ks, vs;
};

template <int D>
__device__ __forceinline__ void load_k(Codes<D>& c, const Cache& cc, int64_t bh, int in, int lane) {
    const int8_t* base = cc.k + (bh * cc.bs + in) * D + (lane >> 2) * D + (lane & 3) * 16;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int i = 0; i < Codes<D>::KC; ++i) c.k[nt][i] = ld_code16(base + nt * 8 * D + i * 64);
    c.ks = __ldg(cc.ks + bh);
}
template <int D>
__device__ __forceinline__ void load_v(Codes<D>& c, const Cache& cc, int64_t bh, int in, int lane) {
    const int g = lane >> 2, q = lane & 3;
    const int8_t* base = cc.v + (bh * cc.bs + in) * D;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int8_t* row = base + (2 * q + (t & 1) + (t >> 1) * 8) * D;
        if constexpr (D == 64) {
            const uint2 w = ld_code8(row + g * 8);
            c.v[t][0] = make_uint4(w.x, w.y, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < Codes<D>::VC; ++i) c.v[t][i] = ld_code16(row + i * 128 + g * 16);
        }
    }
    c.vs = __ldg(cc.vs + bh);
}

constexpr float kShift = 15.0f;  // a step's weights are exp2(x - largest of the step + 15): at most 2^15, and fp16 keeps
                                 // 11 bits of those down to 2^-29 of the step's largest
constexpr float kLazy = 40.0f;   // a row's reference m moves when a step exceeds it by 2^40: fp32 holds the sums until then

// The tile's rows against steps first + off, first + off + stride, ... below first + n of request r's keys and values.
// Per step of 16 tokens: x = q . k (fp16 products of exact codes, fp32 sums) times the block's key scale; weights
// exp2(x - the row's largest x of the step); the row's sum l and outputs o in fp32 relative to exp2(m), m one of the
// rows' earlier maxima: o = o + exp2(step's largest - m) * (block's value scale) * (weights . codes), where the product
// of a step starts from zero, so the factors of a step are applied in fp32.  Weights enter the product as one fp16
// value (SP 1: 2^-12 of each, averaged over the tokens, for 16-bit outputs) or as two (SP 2).
// The next step's keys are loaded as soon as this step's are used, its values likewise, so that half of a step's
// bytes are in flight at any time without a second set of registers.
template <int D, int SP>
__device__ __forceinline__ void attend(const AttnParams& p, const uint4* qf, const float* rowf, const Req& q, int r, int h,
                                       int rt, int first, int n, int off, int stride, Rows<D>& R, int lane) {
    const int g = lane >> 2, qd = lane & 3;
    const int32_t* tab = p.table + (int64_t) r * p.table_stride;
    const int per = p.c.bs / kStep;
    int pos[2], low[2];              // a row sees the keys low .. pos
    int pmin = INT_MAX, lmax = INT_MIN;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = rt * 16 + g + 8 * i, rows = q.n * p.G;
        pos[i] = q.len - q.n + min(row, rows - 1) / p.G;
        low[i] = p.window > 0 ? pos[i] - p.window + 1 : INT_MIN;
    }
    {
        const int rows = q.n * p.G;
        pmin = q.len - q.n + (rt * 16) / p.G;
        const int pmax = q.len - q.n + (min(rt * 16 + 16, rows) - 1) / p.G;
        lmax = p.window > 0 ? pmax - p.window + 1 : INT_MIN;
    }
    const float rf[2] = {rowf[g], rowf[g + 8]};
    auto block = [&](int s) -> int {
        const int b = s < n ? __ldg(tab + (first + s) / per) : -1;
        return b < p.c.n_blocks ? b : -1;
    };
    Codes<D> c;
    int s = off;
    int id = block(s), id_next = block(s + stride);
    if (id >= 0) {
        const int64_t bh = (int64_t) id * p.c.H + h;
        load_k<D>(c, p.c, bh, (first + s) % per * kStep, lane);
        load_v<D>(c, p.c, bh, (first + s) % per * kStep, lane);
    }
    for (; s < n; s += stride) {
        const int id_after = block(s + 2 * stride);
        const int in_next = (first + s + stride) % per * kStep;
        const int64_t bh_next = (int64_t) id_next * p.c.H + h;
        float x[2][4];
        if (id >= 0) {
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) x[nt][0] = x[nt][1] = x[nt][2] = x[nt][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < Codes<D>::KC; ++i) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    const uint4 a4 = qf[(i * 4 + kk) * 32 + lane];
                    const uint32_t a[4] = {a4.x, a4.y, a4.z, a4.w};
                    uint32_t b[4] = {0, 0, 0, 0};
                    if (SP == 2) {
                        const uint4 b4 = qf[(D / 16 + i * 4 + kk) * 32 + lane];
                        b[0] = b4.x, b[1] = b4.y, b[2] = b4.z, b[3] = b4.w;
                    }
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        const uint32_t w = (kk == 0 ? c.k[nt][i].x : kk == 1 ? c.k[nt][i].y : kk == 2 ? c.k[nt][i].z : c.k[nt][i].w) ^ 0x80808080u;
                        const uint32_t b0 = half_pair(w, 0x4140), b1 = half_pair(w, 0x4342);
                        mma_f16(x[nt], a, b0, b1);
                        if (SP == 2) mma_f16(x[nt], b, b0, b1);
                    }
                }
            }
        }
        const float ks = c.ks;
        if (id_next >= 0) load_k<D>(c, p.c, bh_next, in_next, lane);
        if (id >= 0) {
            const int t0 = (first + s) * kStep;
            const bool edge = t0 + kStep - 1 > pmin || t0 < lmax;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = e >> 1, t = t0 + nt * 8 + 2 * qd + (e & 1);
                    x[nt][e] *= ks * rf[i];
                    if (edge && (t > pos[i] || t < low[i])) x[nt][e] = -INFINITY;
                }
            float mx[2], al[2], f[2];
            bool moved = false;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                mx[i] = fmaxf(fmaxf(x[0][2 * i], x[0][2 * i + 1]), fmaxf(x[1][2 * i], x[1][2 * i + 1]));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                al[i] = 1.0f;
                if (mx[i] > R.m[i] + kLazy) {        // true for the first key of a row (m = -inf)
                    al[i] = ex2(R.m[i] - mx[i]);
                    R.m[i] = mx[i];
                    moved = true;
                }
                f[i] = mx[i] == -INFINITY ? 0.0f : ex2(mx[i] - R.m[i]);
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int j = 0; j < D / 8; ++j) {
                    R.o[j][0] *= al[0], R.o[j][1] *= al[0];
                    R.o[j][2] *= al[1], R.o[j][3] *= al[1];
                }
                R.l[0] *= al[0], R.l[1] *= al[1];
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float z = mx[i] == -INFINITY ? 0.0f : mx[i] - kShift;
                float sum = 0.0f;
#pragma unroll
                for (int nt = 0; nt < 2; ++nt) {
                    const float p0 = ex2(x[nt][2 * i] - z), p1 = ex2(x[nt][2 * i + 1] - z);
                    sum += p0 + p1;
                    const uint32_t u = pack_f16(p0, p1);
                    hi[nt * 2 + i] = u;
                    if (SP == 2) {
                        const float2 w = __half22float2(*(const __half2*) &u);
                        lo[nt * 2 + i] = pack_f16(p0 - w.x, p1 - w.y);
                    }
                }
                R.l[i] = fmaf(sum, f[i], R.l[i]);
            }
            f[0] *= c.vs, f[1] *= c.vs;
#pragma unroll
            for (int i = 0; i < Codes<D>::VC; ++i) {
#pragma unroll
                for (int w = 0; w < (D == 64 ? 2 : 4); ++w) {
                    uint32_t y[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        y[t] = (w == 0 ? c.v[t][i].x : w == 1 ? c.v[t][i].y : w == 2 ? c.v[t][i].z : c.v[t][i].w) ^ 0x80808080u;
                    const uint32_t a01 = __byte_perm(y[0], y[1], 0x5140), a23 = __byte_perm(y[0], y[1], 0x7362);
                    const uint32_t b01 = __byte_perm(y[2], y[3], 0x5140), b23 = __byte_perm(y[2], y[3], 0x7362);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t sel = j & 1 ? 0x4342 : 0x4140;
                        const uint32_t b0 = half_pair(j < 2 ? a01 : a23, sel), b1 = half_pair(j < 2 ? b01 : b23, sel);
                        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_f16(acc, hi, b0, b1);
                        if (SP == 2) mma_f16(acc, lo, b0, b1);
                        float* o = R.o[(i * 4 + w) * 4 + j];
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] = fmaf(f[e >> 1], acc[e], o[e]);
                    }
                }
            }
        }
        if (id_next >= 0) load_v<D>(c, p.c, bh_next, in_next, lane);
        id = id_next;
        id_next = id_after;
    }
    // every lane of a row's four holds a part of its sum
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        R.l[i] += __shfl_xor_sync(0xffffffffu, R.l[i], 1);
        R.l[i] += __shfl_xor_sync(0xffffffffu, R.l[i], 2);
    }
}

// Output tile j of a lane holds the columns col(j), col(j) + CW (its two accumulator columns); consecutive j are
// consecutive columns, so a lane's 16 (D = 64: 8) values of a row half are consecutive.
template <int D>
__device__ __forceinline__ int out_col(int j, int half, int qd) {
    constexpr int W = D == 64 ? 8 : 16;
    return (j / W) * 128 + (2 * qd + half) * W + j % W;
}

template <int D>
__device__ __forceinline__ void write_rows(const AttnParams& p, const Req& q, int h, int rt, const Rows<D>& R, int lane) {
    const int g = lane >> 2, qd = lane & 3, rows = q.n * p.G;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = rt * 16 + g + 8 * i;
        if (row >= rows) continue;
        const float inv = R.l[i] > 0.0f ? 1.0f / R.l[i] : 0.0f;      // a row that sees no key is zero
        const int64_t base = (int64_t) (q.tok + row / p.G) * p.o_tok + (int64_t) (h * p.G + row % p.G) * p.o_head;
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < D / 8; ++j)
                store_elem(p.o, base + out_col<D>(j, half, qd), p.type, R.o[j][2 * i + half] * inv);
    }
}

// The steps of all (request, head, tile) segments, one after the other (request, then head, then tile), are cut into
// equal ranges, one per CTA; a range's warps take its steps in turn and join their rows through shared memory at the
// end of each segment.  A segment inside one range is finished there; one cut by a range's end leaves its rows, maxima
// and sums for k_attn_join.  So a lone request of 131,072 tokens and 64 requests of uneven lengths fill the GPU alike.
template <int D, int SP>
__global__ void __launch_bounds__(kAttnWarps * 32) k_attn_split(const AttnParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    uint4* qf = (uint4*) smem;                                         // [SP][D / 16][32]
    float* mrg = (float*) (smem + SP * (D / 16) * 32 * 16);            // [2][16][D] rows in transit between warps
    float* ml = mrg + 2 * 16 * D;                                      // [2][2][16]
    float* rowf = ml + 64;                                             // [16]
    int64_t* pre = (int64_t*) (rowf + 16);                             // [n_req + 1]
    __shared__ int64_t wsum[kAttnWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int R = p.n_req, T = kAttnWarps * 32;
    // steps before each request
    {
        const int per = (R + T - 1) / T, r0 = min(tid * per, R), r1 = min(r0 + per, R);
        int64_t sum = 0;
        for (int r = r0; r < r1; ++r) {
            const Req q = attn_req(p, r);
            for (int rt = 0; rt < p.tiles; ++rt) {
                int f, n;
                tile_steps(p, q, rt, f, n);
                sum += (int64_t) n * p.c.H;
            }
        }
        int64_t v = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += u;
        }
        if (lane == 31) wsum[warp] = v;
        __syncthreads();
        int64_t x = v - sum;
        for (int w = 0; w < warp; ++w) x += wsum[w];
        for (int r = r0; r < r1; ++r) {
            pre[r] = x;
            const Req q = attn_req(p, r);
            for (int rt = 0; rt < p.tiles; ++rt) {
                int f, n;
                tile_steps(p, q, rt, f, n);
                x += (int64_t) n * p.c.H;
            }
        }
        if (tid == T - 1) pre[R] = x;
        __syncthreads();
    }
    if (blockIdx.x == 0)
        for (int r = tid; r <= R; r += T) p.pre[r] = pre[r];
    const int64_t total = pre[R];
    const int64_t per_cta = max((int64_t) (2 * kAttnWarps), (total + gridDim.x - 1) / gridDim.x);
    const int64_t begin = (int64_t) blockIdx.x * per_cta, end = min(begin + per_cta, total);
    if (begin >= end) return;
    int r = 0;
    {
        int lo = 0, hi = R - 1;                       // the last request with pre[r] <= begin
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pre[mid] <= begin) lo = mid;
            else hi = mid - 1;
        }
        r = lo;
    }
    for (int64_t at = begin; at < end;) {
        while (pre[r + 1] <= at) ++r;
        const Req q = attn_req(p, r);
        const int64_t all = (pre[r + 1] - pre[r]) / p.c.H;        // steps of one head
        const int h = (int) ((at - pre[r]) / all);
        int64_t in = (at - pre[r]) - (int64_t) h * all;
        int rt = 0, first = 0, n = 0;
        for (;; ++rt) {
            tile_steps(p, q, rt, first, n);
            if (in < n) break;
            in -= n;
        }
        const int64_t seg = at - in;                              // where the segment starts
        const int take = (int) min((int64_t) n - in, end - at);
        stage_rows<D, SP>(p, q, h, rt, qf, rowf, warp, kAttnWarps, lane);
        __syncthreads();
        Rows<D> rows;
        rows.clear();
        attend<D, SP>(p, qf, rowf, q, r, h, rt, first + (int) in, take, warp, kAttnWarps, rows, lane);
        const int g = lane >> 2, qd = lane & 3;
#pragma unroll
        for (int half_w = kAttnWarps / 2; half_w; half_w /= 2) {
            if (warp >= half_w && warp < 2 * half_w) {
                float* b = mrg + (warp - half_w) * 16 * D;
#pragma unroll
                for (int j = 0; j < D / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) b[(j * 4 + e) * 32 + lane] = rows.o[j][e];
                if (qd == 0) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        ml[(warp - half_w) * 32 + g + 8 * i] = rows.m[i];
                        ml[(warp - half_w) * 32 + 16 + g + 8 * i] = rows.l[i];
                    }
                }
            }
            __syncthreads();
            if (warp < half_w) {
                const float* b = mrg + warp * 16 * D;
                float fa[2], fb[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float mb = ml[warp * 32 + g + 8 * i], lb = ml[warp * 32 + 16 + g + 8 * i];
                    const float m = fmaxf(rows.m[i], mb);
                    fa[i] = rows.m[i] == -INFINITY ? 0.0f : ex2(rows.m[i] - m);
                    fb[i] = mb == -INFINITY ? 0.0f : ex2(mb - m);
                    rows.m[i] = m;
                    rows.l[i] = rows.l[i] * fa[i] + lb * fb[i];
                }
#pragma unroll
                for (int j = 0; j < D / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        rows.o[j][e] = rows.o[j][e] * fa[e >> 1] + b[(j * 4 + e) * 32 + lane] * fb[e >> 1];
            }
            __syncthreads();
        }
        if (warp == 0) {
            if (take == n) {
                write_rows<D>(p, q, h, rt, rows, lane);
            } else {
                const int64_t slot = 2 * (int64_t) blockIdx.x + (seg > begin ? 1 : 0);
                float* b = p.part + slot * 16 * D;
                float* s = p.part + 2 * (int64_t) p.n_cta * 16 * D + slot * 32;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int half = 0; half < 2; ++half)
#pragma unroll
                        for (int j = 0; j < D / 8; j += 4)
                            *(float4*) (b + (g + 8 * i) * D + out_col<D>(j, half, qd)) =
                                make_float4(rows.o[j][2 * i + half], rows.o[j + 1][2 * i + half], rows.o[j + 2][2 * i + half],
                                            rows.o[j + 3][2 * i + half]);
                    if (qd == 0) s[g + 8 * i] = rows.m[i], s[16 + g + 8 * i] = rows.l[i];
                }
            }
        }
        at += take;
    }
}

// One warp per (request, head, tile) row: the rows of the ranges that a segment was cut into, joined by their maxima;
// zeros for a row of a segment without keys.  Segments inside one range were finished by k_attn_split.
template <int D>
__global__ void __launch_bounds__(128) k_attn_join(const AttnParams p) {
    const int lane = threadIdx.x & 31;
    const int seg_id = blockIdx.x, i = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int rt = seg_id % p.tiles, h = seg_id / p.tiles % p.c.H, r = seg_id / p.tiles / p.c.H;
    const Req q = attn_req(p, r);
    const int row = rt * 16 + i;
    if (row >= q.n * p.G) return;
    int first, n;
    const int64_t total = p.pre[p.n_req];
    const int64_t per_cta = max((int64_t) (2 * kAttnWarps), (total + p.n_cta - 1) / p.n_cta);
    int64_t seg = p.pre[r] + (p.pre[r + 1] - p.pre[r]) / p.c.H * h;
    for (int t = 0; t < rt; ++t) {
        tile_steps(p, q, t, first, n);
        seg += n;
    }
    tile_steps(p, q, rt, first, n);
    const int64_t out = (int64_t) (q.tok + row / p.G) * p.o_tok + (int64_t) (h * p.G + row % p.G) * p.o_head;
    if (n == 0) {
        for (int d = lane; d < D; d += 32) store_elem(p.o, out + d, p.type, 0.0f);
        return;
    }
    const int64_t c0 = seg / per_cta, c1 = (seg + n - 1) / per_cta;
    if (c0 == c1) return;
    const float* stats = p.part + 2 * (int64_t) p.n_cta * 16 * D;
    auto slot = [&](int64_t c) { return 2 * c + (seg > c * per_cta ? 1 : 0); };
    float m = -INFINITY;
    for (int64_t c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, stats[slot(c) * 32 + i]);
    m = warp_max(m);
    float acc[D / 32], l = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) acc[j] = 0.0f;
#pragma unroll 4
    for (int64_t c = c0; c <= c1; ++c) {
        const float mc = stats[slot(c) * 32 + i], lc = stats[slot(c) * 32 + 16 + i];
        const float f = mc == -INFINITY ? 0.0f : ex2(mc - m);
        const float* b = p.part + (slot(c) * 16 + i) * D;
        l = fmaf(lc, f, l);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) acc[j] = fmaf(b[j * 32 + lane], f, acc[j]);
    }
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) store_elem(p.o, out + j * 32 + lane, p.type, acc[j] * inv);
}

// Many rows: one warp per 16-row tile, every step of the tile by the same warp; the four warps of a CTA take
// neighbouring tiles of a head, so they share the codes through the caches.
template <int D, int SP>
__global__ void __launch_bounds__(kAttnWarps * 32) k_attn_tiles(const AttnParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint4* qf = (uint4*) smem + warp * SP * (D / 16) * 32;
    float* rowf = (float*) ((uint4*) smem + kAttnWarps * SP * (D / 16) * 32) + warp * 16;
    const int rt = (gridDim.x - 1 - blockIdx.x) * kAttnWarps + warp, h = blockIdx.y, r = blockIdx.z;
    const Req q = attn_req(p, r);
    if (rt * 16 >= q.n * p.G) return;
    stage_rows<D, SP>(p, q, h, rt, qf, rowf, 0, 1, lane);
    __syncwarp();
    int first, n;
    tile_steps(p, q, rt, first, n);
    Rows<D> rows;
    rows.clear();
    attend<D, SP>(p, qf, rowf, q, r, h, rt, first, n, 0, 1, rows, lane);
    write_rows<D>(p, q, h, rt, rows, lane);
}

// ------------------------------------------------------------------------------------------------ host
int check_cache(const tsb_kv8* c, const char* what) {
    if (!c || c->struct_size != sizeof(tsb_kv8)) return cfail(TSB_ERR_ARG, "%s: cache struct_size", what);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || c->n_blocks < 1 || c->n_kv_heads < 1)
        return cfail(TSB_ERR_ARG, "%s: cache pointers and sizes", what);
    if (c->block_size != 16 && c->block_size != 32 && c->block_size != 64)
        return cfail(TSB_ERR_UNSUPPORTED, "%s: block_size %d (16, 32 or 64)", what, c->block_size);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return cfail(TSB_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128 or 256)", what, c->head_dim);
    if ((uintptr_t) c->k % 16 || (uintptr_t) c->v % 16 || (uintptr_t) c->k_scale % 4 || (uintptr_t) c->v_scale % 4)
        return cfail(TSB_ERR_ALIGN, "%s: the code pools must be 16-byte aligned", what);
    return TSB_OK;
}
Cache cache_of(const tsb_kv8* c) {
    return Cache{c->k, c->v, c->k_scale, c->v_scale, c->n_blocks, c->block_size, c->n_kv_heads, c->head_dim};
}
bool elem_ok(int t) { return t == E_F32 || t == E_F16 || t == E_BF16; }

struct AttnPlan {
    int G, tiles, n_cta;
    bool split;
    uint64_t ws;
};
int attn_plan(const tsb_kv8* c, const tsb_kv8_attn* d, AttnPlan& a) {
    if (int rc = check_cache(c, "kv8_attention")) return rc;
    if (!d || d->struct_size != sizeof(tsb_kv8_attn)) return cfail(TSB_ERR_ARG, "kv8_attention: struct_size");
    if (!elem_ok(d->elem_type)) return cfail(TSB_ERR_UNSUPPORTED, "kv8_attention: element type %d (F32, F16, BF16)", d->elem_type);
    if (d->n_req < 0 || d->max_q < 0 || d->table_width < 0 || d->window < 0 || d->n_tok < 0)
        return cfail(TSB_ERR_ARG, "kv8_attention: negative sizes");
    if (d->n_req > kMaxReq) return cfail(TSB_ERR_UNSUPPORTED, "kv8_attention: at most %d requests", kMaxReq);
    if (d->q_heads < 1 || d->q_heads % c->n_kv_heads)
        return cfail(TSB_ERR_ARG, "kv8_attention: q_heads %d not a multiple of the cache's %d heads", d->q_heads, c->n_kv_heads);
    if ((int64_t) d->table_width * c->block_size > 0x7fffffffll - 64 || c->n_kv_heads > 65535)
        return cfail(TSB_ERR_UNSUPPORTED, "kv8_attention: at most 2^31 tokens a request and 65535 heads");
    a.G = d->q_heads / c->n_kv_heads;
    const int64_t rows = (int64_t) d->max_q * a.G;
    if (rows > (1 << 28)) return cfail(TSB_ERR_UNSUPPORTED, "kv8_attention: too many query rows");
    a.tiles = (int) ((rows + 15) / 16);
    a.split = rows <= kSplitRows;
    const int sms = sm_count();
    if (!sms) return cfail(TSB_ERR_CUDA, "kv8_attention: no CUDA device");
    a.n_cta = sms * (c->head_dim == 256 ? 2 : c->head_dim == 128 ? 3 : 4);
    a.ws = a.split ? (((uint64_t) d->n_req + 1) * 8 + 255) / 256 * 256 + (uint64_t) a.n_cta * 2 * (16 * c->head_dim + 32) * 4 : 0;
    return TSB_OK;
}

template <int D, int SP>
int launch_attn(const AttnParams& p, const AttnPlan& a, cudaStream_t st) {
    const int qf = SP * (D / 16) * 32 * 16;
    if (a.split) {
        const int sm = qf + 2 * 16 * D * 4 + 64 * 4 + 16 * 4 + (p.n_req + 1) * 8;
        if (sm > 48 * 1024 &&
            cudaFuncSetAttribute(k_attn_split<D, SP>, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) != cudaSuccess)
            return ccuda("kv8_attention: shared memory");
        k_attn_split<D, SP><<<a.n_cta, kAttnWarps * 32, sm, st>>>(p);
        k_attn_join<D><<<dim3((unsigned) (p.n_req * p.c.H * p.tiles), 4), 128, 0, st>>>(p);
    } else {
        const int sm = kAttnWarps * (qf + 64);
        if (sm > 48 * 1024 &&
            cudaFuncSetAttribute(k_attn_tiles<D, SP>, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) != cudaSuccess)
            return ccuda("kv8_attention: shared memory");
        k_attn_tiles<D, SP><<<dim3((unsigned) ((p.tiles + kAttnWarps - 1) / kAttnWarps), p.c.H, p.n_req), kAttnWarps * 32, sm, st>>>(p);
    }
    return ccuda("kv8_attention");
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" {

int tsb_block_tables(const int32_t* lens, const int32_t* n_new, const uint8_t* done, int n_req, int32_t* table,
                     int64_t table_stride, int table_width, int32_t* free_list, int free_cap, const int32_t* n_free,
                     int block_size, int32_t* lens_out, int32_t* cu_new, int64_t* slots, int64_t cap_tokens,
                     int32_t* n_free_out, void* stream) {
    if (n_req < 0 || table_width < 0 || free_cap < 0 || block_size < 1 || cap_tokens < 0)
        return cfail(TSB_ERR_ARG, "block_tables: negative sizes");
    if (n_req > kTabMaxReq) return cfail(TSB_ERR_UNSUPPORTED, "block_tables: at most %d requests", kTabMaxReq);
    if ((n_req && (!lens || !n_new || !table || !lens_out)) || !n_free || !n_free_out || !cu_new || (free_cap && !free_list) ||
        (cap_tokens && !slots))
        return cfail(TSB_ERR_ARG, "block_tables: null pointer");
    if (table_stride < table_width) return cfail(TSB_ERR_ARG, "block_tables: table_stride");
    if (n_free == n_free_out || (n_req && lens == lens_out))
        return cfail(TSB_ERR_ARG, "block_tables: lens_out and n_free_out must not be the inputs (every CTA reads those)");
    const TabParams p{lens, n_new, done, n_req, table, table_stride, table_width, free_list, free_cap, n_free, block_size,
                      lens_out, cu_new, slots, cap_tokens, n_free_out};
    const int sm = 3 * (n_req + 1) * 4;
    if (sm > 47 * 1024 &&
        cudaFuncSetAttribute(k_block_tables, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) != cudaSuccess)
        return ccuda("block_tables: shared memory");
    const int64_t work = std::max<int64_t>(cap_tokens, n_req);
    const int ctas = (int) std::min<int64_t>(std::max<int64_t>((work + kTabThreads - 1) / kTabThreads, 1), std::max(sm_count(), 1));
    k_block_tables<<<ctas, kTabThreads, sm, cst(stream)>>>(p);
    return ccuda("block_tables");
}

int tsb_kv8_append(const tsb_kv8* cache, const void* k, const void* v, int elem_type, int64_t k_tok, int64_t k_head,
                   int64_t v_tok, int64_t v_head, const int64_t* slots, int64_t n_tok, void* stream) {
    if (int rc = check_cache(cache, "kv8_append")) return rc;
    if (!elem_ok(elem_type)) return cfail(TSB_ERR_UNSUPPORTED, "kv8_append: element type %d (F32, F16, BF16)", elem_type);
    if (n_tok < 0) return cfail(TSB_ERR_ARG, "kv8_append: n_tok");
    if (n_tok == 0) return TSB_OK;
    if (!k || !v || !slots) return cfail(TSB_ERR_ARG, "kv8_append: null pointer");
    const int es = elem_bytes(elem_type);
    if ((uintptr_t) k % es || (uintptr_t) v % es) return cfail(TSB_ERR_ALIGN, "kv8_append: element alignment");
    if (cache->n_kv_heads > 65535) return cfail(TSB_ERR_UNSUPPORTED, "kv8_append: at most 65535 heads");
    AppendParams p{cache_of(cache), k, v, elem_type, k_tok, k_head, v_tok, v_head, slots, n_tok, 0, false};
    p.wide = !((uintptr_t) k % 16 || (uintptr_t) v % 16 || (k_tok * es) % 16 || (k_head * es) % 16 || (v_tok * es) % 16 ||
               (v_head * es) % 16);
    p.per_cta = n_tok <= 1024 ? 4 : 32;
    const int64_t chunks = (n_tok + p.per_cta - 1) / p.per_cta;
    if (chunks > 0x7fffffffll) return cfail(TSB_ERR_UNSUPPORTED, "kv8_append: too many tokens");
    k_kv8_append<<<dim3((unsigned) chunks, cache->n_kv_heads), 256, 0, cst(stream)>>>(p);
    return ccuda("kv8_append");
}

int tsb_kv8_read(const tsb_kv8* cache, const int64_t* slots, int64_t n_tok, void* k, void* v, int elem_type, void* stream) {
    if (int rc = check_cache(cache, "kv8_read")) return rc;
    if (!elem_ok(elem_type)) return cfail(TSB_ERR_UNSUPPORTED, "kv8_read: element type %d (F32, F16, BF16)", elem_type);
    if (n_tok < 0) return cfail(TSB_ERR_ARG, "kv8_read: n_tok");
    if (n_tok == 0) return TSB_OK;
    if (!k || !v || !slots) return cfail(TSB_ERR_ARG, "kv8_read: null pointer");
    if ((uintptr_t) k % 16 || (uintptr_t) v % 16) return cfail(TSB_ERR_ALIGN, "kv8_read: 16-byte aligned outputs");
    const int64_t n = n_tok * cache->n_kv_heads * (cache->head_dim / 16), ctas = (n + 255) / 256;
    if (ctas > 0x7fffffffll) return cfail(TSB_ERR_UNSUPPORTED, "kv8_read: too many tokens");
    k_kv8_read<<<(unsigned) ctas, 256, 0, cst(stream)>>>(cache_of(cache), slots, n_tok, k, v, elem_type);
    return ccuda("kv8_read");
}

uint64_t tsb_kv8_attention_workspace_bytes(const tsb_kv8* cache, const tsb_kv8_attn* d) {
    AttnPlan a;
    return attn_plan(cache, d, a) == TSB_OK ? a.ws : 0;
}

int tsb_kv8_attention(const tsb_kv8* cache, const tsb_kv8_attn* d, const void* q, const int32_t* table, const int32_t* lens,
                      const int32_t* cu_q, void* out, void* workspace, uint64_t ws_bytes, void* stream) {
    AttnPlan a;
    if (int rc = attn_plan(cache, d, a)) return rc;
    if (d->n_req == 0 || d->n_tok == 0 || d->max_q == 0) return TSB_OK;
    if (!q || !out || !lens || (!table && d->table_width)) return cfail(TSB_ERR_ARG, "kv8_attention: null pointer");
    if (!cu_q && d->n_tok < (int64_t) d->n_req * d->max_q)
        return cfail(TSB_ERR_ARG, "kv8_attention: without cu_q every request has max_q queries");
    if (d->table_stride < d->table_width) return cfail(TSB_ERR_ARG, "kv8_attention: table_stride");
    const int es = elem_bytes(d->elem_type);
    if ((uintptr_t) q % es || (uintptr_t) out % es) return cfail(TSB_ERR_ALIGN, "kv8_attention: element alignment");
    if (a.ws && (!workspace || ws_bytes < a.ws))
        return cfail(TSB_ERR_WORKSPACE, "kv8_attention: workspace of %llu bytes needed", (unsigned long long) a.ws);
    if (a.ws && (uintptr_t) workspace % 16) return cfail(TSB_ERR_ALIGN, "kv8_attention: 16-byte aligned workspace");
    if ((int64_t) d->n_req * cache->n_kv_heads * a.tiles > 0x7fffffffll || d->n_req > 65535)
        return cfail(TSB_ERR_UNSUPPORTED, "kv8_attention: too many requests");
    AttnParams p{};
    p.c = cache_of(cache);
    p.q = q, p.o = out, p.type = d->elem_type, p.n_req = d->n_req, p.G = a.G, p.max_q = d->max_q, p.window = d->window;
    p.scale_log2 = d->scale * 1.4426950408889634f;
    p.q_tok = d->q_tok, p.q_head = d->q_head, p.o_tok = d->o_tok, p.o_head = d->o_head, p.n_tok = d->n_tok;
    p.table = table, p.table_stride = d->table_stride, p.width = d->table_width, p.lens = lens, p.cu = cu_q;
    p.tiles = a.tiles, p.n_cta = a.n_cta;
    p.pre = (int64_t*) workspace;
    p.part = (float*) ((uint8_t*) workspace + (((uint64_t) d->n_req + 1) * 8 + 255) / 256 * 256);
    const bool two = d->elem_type == E_F32;
    cudaStream_t st = cst(stream);
    switch (cache->head_dim) {
        case 64: return two ? launch_attn<64, 2>(p, a, st) : launch_attn<64, 1>(p, a, st);
        case 128: return two ? launch_attn<128, 2>(p, a, st) : launch_attn<128, 1>(p, a, st);
        default: return two ? launch_attn<256, 2>(p, a, st) : launch_attn<256, 1>(p, a, st);
    }
}

}  // extern "C"
