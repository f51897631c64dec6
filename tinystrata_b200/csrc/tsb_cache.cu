// tsb_cache.cu - the paged 8-bit key / value cache of a serving step: block tables and slot maps from the requests'
// lengths, appending and reading back tokens, and attention over the cache.
//
// The cache is two pools of int8 codes [n_blocks][n_kv_heads][block_size][head_dim] with one fp32 scale per (block, head):
// a key or value is code * scale.  The tokens of one (block, head) are contiguous, so a warp that attends 16 tokens
// reads 16 * head_dim consecutive bytes, and every token of such a step shares one scale.
#include "../../include/tsb_moe.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
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

constexpr int kMaxDev = 64;
int device() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDev) {
        cudaGetLastError();
        return -1;
    }
    return dev;
}
}  // namespace
// The current device's multiprocessors, 0 without a device (used by tsb_delta.cu too).
int sm_count() {
    static std::atomic<int> known[kMaxDev];
    const int dev = device();
    if (dev < 0) return 0;
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        known[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}
namespace {
// The most dynamic shared memory that a kernel can ask for, granted once a device.  (Always the same size: the attribute is
// set, not raised, so that two threads with sizes of their own could leave the smaller one.)
template <class K>
int allow_smem(K* kernel, std::atomic<bool> (&granted)[kMaxDev], int most, const char* what) {
    const int dev = device();
    if (dev < 0) return cfail(TSB_ERR_CUDA, "%s: no CUDA device", what);
    if (granted[dev].load(std::memory_order_acquire)) return TSB_OK;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) return ccuda(what);
    granted[dev].store(true, std::memory_order_release);
    return TSB_OK;
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
// Block counts in 32 bits: two lengths sum to less than 2^32.
__device__ __forceinline__ unsigned blocks_of(unsigned n, unsigned bs) { return n ? (n - 1) / bs + 1 : 0; }
__device__ __forceinline__ TabReq tab_req(const TabParams& p, int r) {
    TabReq q;
    q.len = max(p.lens[r], 0);
    q.add = max(p.n_new[r], 0);
    q.done = p.done && p.done[r] != 0;
    q.has = (int) blocks_of(q.len, p.block_size);
    const unsigned after = blocks_of((unsigned) q.len + (unsigned) q.add, p.block_size);
    q.fits = !q.done && after <= (unsigned) p.width;
    q.gives = q.done ? min(q.has, p.width) : 0;
    q.takes = q.fits ? (int) after - q.has : 0;
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
// requests nothing else is left (5.6 us), at 1000 requests and 33,000 tokens the slots' 8 bytes a token are 0.3 MB (9.2 us).
__global__ void __launch_bounds__(kTabThreads) k_block_tables(const TabParams p) {
    extern __shared__ int sh[];
    const int R = p.n_req;
    int* cu = sh;                     // R + 1
    int* take = sh + (R + 1);         // R + 1
    int* give = sh + 2 * (R + 1);     // R + 1
    __shared__ int64_t wsum[3][kTabThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (R + kTabThreads - 1) / kTabThreads;
    const int r0 = min(tid * per, R), r1 = min(r0 + per, R);
    const int held = min(max(*p.n_free, 0), p.cap_free);
    // Sums in 64 bits, stored as at most 2^31 - 1: refused requests count with whatever they ask for, and each prefix has to
    // stay at or above the one before, since the searches below index with their differences.
    int64_t s[3] = {0, 0, 0};
    for (int r = r0; r < r1; ++r) {
        const TabReq q = tab_req(p, r);
        cu[r] = q.add, take[r] = q.takes, give[r] = q.gives;      // this thread's own, sums below
        s[0] += q.add, s[1] += q.takes, s[2] += q.gives;
    }
    int64_t x[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        int64_t v = s[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
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
    auto stored = [](int64_t v) { return (int) min(v, (int64_t) INT32_MAX); };
    for (int r = r0; r < r1; ++r) {
        const int add = cu[r], takes = take[r], gives = give[r];
        cu[r] = stored(x[0]), take[r] = stored(x[1]), give[r] = stored(x[2]);
        x[0] += add, x[1] += takes, x[2] += gives;
    }
    if (tid == kTabThreads - 1) cu[R] = stored(x[0]), take[R] = stored(x[1]), give[R] = stored(x[2]);
    __syncthreads();

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
    for (int64_t i0 = g; i0 < given; i0 += 4 * step) {              // four table reads in flight
        int b[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t i = i0 + u * step;
            if (i >= given) break;
            const int r = last_le(give, R, i);
            b[u] = p.table[(int64_t) r * p.table_stride + (i - give[r])];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + u * step < given) p.free_list[held + i0 + u * step] = b[u];
    }
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
                const unsigned pos = (unsigned) q.len + (unsigned) (t - cu[r]);
                const int j = (int) (pos / (unsigned) p.block_size);
                const int b = j < q.has ? p.table[(int64_t) r * p.table_stride + j]
                                        : stack(have - 1 - (take[r] + (j - q.has)));
                slot = b < 0 ? -1 : (int64_t) b * p.block_size + (pos - (unsigned) j * (unsigned) p.block_size);
            }
        }
        p.slots[t] = slot;
    }
}

// ------------------------------------------------------------------------------------------------ append, read back
struct Cache {
    int8_t *k, *v;
    float *ks, *vs;
    int n_blocks, bs, H, D, shift;   // block_size = 1 << shift
};

struct AppendParams {
    Cache c;
    const void *k, *v;
    int type;
    int64_t k_tok, k_head, v_tok, v_head;
    const int64_t* slots;
    int64_t n_tok;
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

// The largest magnitude bits of values that are stored as they are, for spotting the others (NaN, infinities) at once.
constexpr uint32_t kPlainBits = 0x7f7f0000u;   // the largest finite bf16
__device__ __forceinline__ uint32_t peak_bits(const float (&x)[8], uint32_t m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
    return m;
}
__device__ __forceinline__ float peak_value(float (&x)[8]) {          // and the values as they are stored
    uint32_t m = peak_bits(x, 0);
    if (m > kPlainBits) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = cache_value(x[j]);
        m = peak_bits(x, 0);
    }
    return __uint_as_float(m);
}
// Eight codes of plain values: rint(x / scale) as the division gives it.  The product with the reciprocal is within
// 3 * 2^-24 * 127 of the quotient, so unless it lies that near to half way between two whole numbers both round alike;
// adding 1.5 * 2^23 rounds to even and leaves the code in the low byte.  (The division itself bound the kernel: 82 us
// for 16,024 tokens of 8 heads.)
__device__ __forceinline__ uint2 encode8(const float (&x)[8], float scale, float inv) {
    uint32_t u[2];
    float far = scale > 1e-30f ? 0.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float q = x[4 * i + j] * inv, r = q + 12582912.0f;
            t[j] = __float_as_uint(r);
            far = fmaxf(far, fabsf(q - (r - 12582912.0f)));
        }
        u[i] = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
    }
    if (far > 0.4998f) {
        u[0] = u[1] = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j >> 2] |= (uint32_t) (uint8_t) cache_code(x[j], scale) << (8 * (j & 3));
    }
    return make_uint2(u[0], u[1]);
}

// 16 codes under a scale that grew: ratio = old / new.
__device__ __forceinline__ uint4 rescale_codes(uint4 w, float ratio) {
    uint32_t* u = (uint32_t*) &w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t r = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) r |= (uint32_t) (uint8_t) (int8_t) rintf((float) (int8_t) (u[i] >> (8 * j)) * ratio) << (8 * j);
        u[i] = r;
    }
    return w;
}

// The slots of a token's neighbours, lane by lane: at[..] of token t on, before[..] back from t - 1 (the second 32 in blocks
// of 64; -1 past the ends).
struct Near {
    int64_t at[2], before[2];
};
__device__ __forceinline__ Near near_slots(const AppendParams& p, int64_t t, int lane) {
    Near n;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t up = t + i * 32 + lane, down = t - 1 - i * 32 - lane;
        const bool use = i == 0 || p.c.bs > 32;
        n.at[i] = use && up < p.n_tok ? p.slots[up] : -1;
        n.before[i] = use && down >= 0 ? p.slots[down] : -1;
    }
    return n;
}
// Whether an earlier token of the call is in the block of the token at s: in its place before it, skipped ones between or not.
__device__ __forceinline__ bool follows(const Near& n, int64_t s, int off, int lane) {
    return __any_sync(0xffffffffu, (lane < off && n.before[0] == s - 1 - lane) || (lane + 32 < off && n.before[1] == s - 33 - lane));
}
// The call's tokens in that block from it on: bit i, the token i places after it, at s + i.
__device__ __forceinline__ uint64_t block_tokens(const Near& n, int64_t s, int room, int lane) {
    const unsigned lo = __ballot_sync(0xffffffffu, lane < room && n.at[0] == s + lane);
    const unsigned hi = __ballot_sync(0xffffffffu, lane + 32 < room && n.at[1] == s + 32 + lane);
    return (uint64_t) hi << 32 | lo;
}
// The first run of those tokens, taken out of them: its first place and its length.
__device__ __forceinline__ int next_run(uint64_t& tokens, int& len) {
    const int skip = __ffsll((long long) tokens) - 1;
    const uint64_t rest = tokens >> skip;
    len = rest == ~0ull ? 64 : __ffsll((long long) ~rest) - 1;
    tokens = skip + len < 64 ? tokens >> (skip + len) << (skip + len) : 0;
    return skip;
}

// Warp (keys or values, head, token), for decode steps, where nearly every token is a run of its own.  A run is the tokens
// of one call that follow one another within one cache block; the block's first token is the leader, and its warp takes the
// block's runs, of which there are several only around skipped tokens, one after the other:
// the largest magnitude over it, the block's new scale max(old, largest / 127) (old: none when the run starts the block), the block's earlier codes
// brought to it when it grew, and the run's codes.  One warp owns the (block, head), so no value is written twice and
// nothing is atomic.  Divisions are IEEE: the same codes on any device.  Bound by the chain of loads: slots, rows, scale
// (48 tokens of 2 heads of 256: 3.1 us).
__global__ void __launch_bounds__(128) k_kv8_append(const AppendParams p) {
    const int lane = threadIdx.x & 31;
    const int bs = p.c.bs, D = p.c.D, DV = D / 8, dvs = D == 64 ? 3 : D == 128 ? 4 : 5;
    const int64_t cap = (int64_t) p.c.n_blocks << p.c.shift;
    const unsigned part = blockIdx.x / p.c.H;
    const int h = (int) (blockIdx.x - part * p.c.H);
    const bool is_v = part & 1;
    const int64_t t = (int64_t) (part >> 1) * 4 + (threadIdx.x >> 5);
    if (t >= p.n_tok) return;
    const void* src = is_v ? p.v : p.k;
    const int64_t row = is_v ? p.v_tok : p.k_tok, col = (is_v ? p.v_head : p.k_head) * h;
    const Near near = near_slots(p, t, lane);
    const int64_t s = __shfl_sync(0xffffffffu, near.at[0], 0), blk = s >> p.c.shift;
    const int at = (int) (s & (bs - 1));
    if (s < 0 || s >= cap || follows(near, s, at, lane)) return;
    int8_t* codes = (is_v ? p.c.v : p.c.k) + ((blk * p.c.H + h) << p.c.shift) * D;
    float* sp = (is_v ? p.c.vs : p.c.ks) + blk * p.c.H + h;
    for (uint64_t todo = block_tokens(near, s, bs - at, lane); todo;) {
        int n;
        const int skip = next_run(todo, n), off = at + skip;
        const int64_t t0 = t + skip;
        const float was = off > 0 ? *sp : 0.0f;
        float peak = 0.0f;
#pragma unroll 4
        for (int e = lane; e < n * DV; e += 32) {
            float x[8];
            load8(x, src, (t0 + (e >> dvs)) * row + col + (e & (DV - 1)) * 8, p.type, p.wide);
            peak = fmaxf(peak, peak_value(x));
        }
        peak = warp_max(peak);
        const float now = fmaxf(was, peak / kCodeMax), inv = 1.0f / now;
        __syncwarp();
        if (lane == 0) *sp = now;
        if (off > 0 && now != was) {
            const float ratio = was / now;
            for (int e = lane; e < off * D / 16; e += 32) ((uint4*) codes)[e] = rescale_codes(((const uint4*) codes)[e], ratio);
        }
#pragma unroll 4
        for (int e = lane; e < n * DV; e += 32) {
            float x[8];
            load8(x, src, (t0 + (e >> dvs)) * row + col + (e & (DV - 1)) * 8, p.type, p.wide);
            peak_value(x);
            *(uint2*) (codes + (int64_t) off * D + (int64_t) e * 8) = encode8(x, now, inv);
        }
        __syncwarp();                                    // the next run reads the scale and the codes
    }
}

// The same for prompts: CTA (chunk of block_size tokens, head, keys or values), the run's values in registers between the
// two passes (up to 64 a thread; a warp's two passes over 16 KB went to memory twice: 82 us for 16,024 tokens of 8 heads).
// Now 61 us for those in fp32, 164 MB, 2.7 TB/s: the latency of load, maximum and codes one after the other at 20 warps a SM
// (issue slots 46% active; a warp waits 2.1 cycles an instruction for its own results, 2.0 for memory, 1.8 for instructions).
__global__ void __launch_bounds__(128, 5) k_kv8_append_runs(const AppendParams p) {
    __shared__ float peaks[4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bs = p.c.bs, D = p.c.D, DV = D / 8, dvs = D == 64 ? 3 : D == 128 ? 4 : 5;
    const int64_t cap = (int64_t) p.c.n_blocks << p.c.shift;
    // heads vary fastest: neighbouring CTAs read a token's whole row
    const unsigned part = blockIdx.x / p.c.H;
    const int h = (int) (blockIdx.x - part * p.c.H);
    const bool is_v = part & 1;
    const int64_t start = (int64_t) (part >> 1) * bs, end_t = min(start + bs, p.n_tok);
    const void* src = is_v ? p.v : p.k;
    const int64_t row = is_v ? p.v_tok : p.k_tok, col = (is_v ? p.v_head : p.k_head) * h;
    for (int64_t base_t = start; base_t < end_t; base_t += 32) {          // every warp finds the leaders for itself
        const int64_t mine = base_t + lane;
        bool leads = false;
        int64_t slot = -1;
        if (mine < end_t) {
            slot = p.slots[mine];
            const int64_t before = mine ? p.slots[mine - 1] : -2;
            leads = slot >= 0 && slot < cap && ((slot & (bs - 1)) == 0 || before != slot - 1);
        }
        for (unsigned todo = __ballot_sync(0xffffffffu, leads); todo; todo &= todo - 1) {
            const int64_t first = base_t + __ffs(todo) - 1;
            const int64_t s = __shfl_sync(0xffffffffu, slot, __ffs(todo) - 1), blk = s >> p.c.shift;
            const int place = (int) (s & (bs - 1));
            const Near near = near_slots(p, first, lane);
            if (place > 1 && follows(near, s, place, lane)) continue;
            int8_t* codes = (is_v ? p.c.v : p.c.k) + ((blk * p.c.H + h) << p.c.shift) * D;
            float* sp = (is_v ? p.c.vs : p.c.ks) + blk * p.c.H + h;
            for (uint64_t runs = block_tokens(near, s, bs - place, lane); runs;) {
                int n;
                const int skip = next_run(runs, n), off = place + skip;
                const int64_t t = first + skip;
                const float was = off > 0 ? *sp : 0.0f;
                constexpr int HOLD = 8;
                float x[HOLD][8], peak = 0.0f;
                auto at = [&](int e) { return (t + (e >> dvs)) * row + col + (e & (DV - 1)) * 8; };
#pragma unroll
                for (int i = 0; i < HOLD; ++i) {
                    const int e = i * 128 + tid;
                    if (e < n * DV) load8(x[i], src, at(e), p.type, p.wide);
                }
#pragma unroll
                for (int i = 0; i < HOLD; ++i) {
                    if (i * 128 + tid >= n * DV) break;
                    peak = fmaxf(peak, peak_value(x[i]));
                }
                for (int e = HOLD * 128 + tid; e < n * DV; e += 128) {         // longer runs: the rest is read twice
                    float y[8];
                    load8(y, src, at(e), p.type, p.wide);
                    peak = fmaxf(peak, peak_value(y));
                }
                peak = warp_max(peak);
                if (lane == 0) peaks[warp] = peak;
                __syncthreads();                                               // also: every thread has read the old scale
                peak = fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3]));
                const float now = fmaxf(was, peak / kCodeMax), inv = 1.0f / now;
                if (tid == 0) *sp = now;
                if (off > 0 && now != was) {
                    const float ratio = was / now;
                    for (int e = tid; e < off * D / 16; e += 128) ((uint4*) codes)[e] = rescale_codes(((const uint4*) codes)[e], ratio);
                }
                auto put = [&](int e, const float (&y)[8]) {
                    *(uint2*) (codes + (int64_t) off * D + (int64_t) e * 8) = encode8(y, now, inv);
                };
#pragma unroll
                for (int i = 0; i < HOLD; ++i) {
                    const int e = i * 128 + tid;
                    if (e < n * DV) put(e, x[i]);
                }
                for (int e = HOLD * 128 + tid; e < n * DV; e += 128) {
                    float y[8];
                    load8(y, src, at(e), p.type, p.wide);
                    peak_value(y);
                    put(e, y);
                }
                __syncthreads();                                               // peaks are read
            }
        }
    }
}

// CTA (share of the tokens, head, keys or values): four codes a thread and step, so that a warp's stores of 16 (8) bytes a
// lane are consecutive, eight steps in flight.  A slot outside the cache reads as zeros.  Bound by latency, slot after slot to
// codes and scale: 16,024 tokens of 8 heads of 128 to fp32 (164 MB) take 45 us, 3.7 TB/s, with the issue slots 42% active and
// a warp waiting 11.6 cycles an instruction for memory.
constexpr int kReadSteps = 8;
__global__ void __launch_bounds__(256) k_kv8_read(const Cache c, const int64_t* __restrict__ slots, int64_t n_tok,
                                                  void* k, void* v, int type) {
    const int per = c.D / 4, ps = c.D == 64 ? 4 : c.D == 128 ? 5 : 6;
    const unsigned share = blockIdx.x / c.H;             // heads vary fastest, as the outputs' rows do
    const int h = (int) (blockIdx.x - share * c.H);
    const bool is_v = share & 1;
    const int8_t* codes = is_v ? c.v : c.k;
    const float* scales = is_v ? c.vs : c.ks;
    void* out = is_v ? v : k;
    const int64_t cap = (int64_t) c.n_blocks << c.shift;
    const int64_t e0 = (int64_t) (share >> 1) * 256 * kReadSteps + threadIdx.x;
    uint32_t w[kReadSteps];
    float sc[kReadSteps];
#pragma unroll
    for (int i = 0; i < kReadSteps; ++i) {
        const int64_t e = e0 + i * 256, t = e >> ps;
        w[i] = 0, sc[i] = 0.0f;
        if (t >= n_tok) continue;
        const int64_t s = slots[t];
        if (s < 0 || s >= cap) continue;
        const int64_t bh = (s >> c.shift) * c.H + h;
        w[i] = *(const uint32_t*) (codes + ((bh << c.shift) + (s & (c.bs - 1))) * c.D + (e & (per - 1)) * 4);
        sc[i] = scales[bh];
    }
#pragma unroll
    for (int i = 0; i < kReadSteps; ++i) {
        const int64_t e = e0 + i * 256, t = e >> ps;
        if (t >= n_tok) break;
        const int64_t at = (t * c.H + h) * c.D + (e & (per - 1)) * 4;
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = (float) (int8_t) (w[i] >> (8 * j)) * sc[i];
        if (type == E_F32) *(float4*) ((float*) out + at) = make_float4(f[0], f[1], f[2], f[3]);
        else if (type == E_F16) *(uint2*) ((uint16_t*) out + at) = make_uint2(pack_f16(f[0], f[1]), pack_f16(f[2], f[3]));
        else *(uint2*) ((uint16_t*) out + at) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
    }
}

// ------------------------------------------------------------------------------------------------ attention
constexpr int kAttnWarps = 4;
constexpr int kStep = 16;            // tokens of a step: one matrix-product depth, always within one cache block
constexpr int kSplitRows = 64, kPromptCtas = 12, kPromptCtas32 = 40;   // see attn_plan
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
    int tiles;                       // row tiles of the longest request
    // split over CTAs: steps before each request, partial rows
    int64_t* pre;                    // [n_req + 1]
    float* part;                     // [2 * CTAs][tile rows][D], then their maxima and sums [2 * CTAs][2][tile rows]
    int n_cta;
    bool wide_out;                   // 16-byte aligned output rows
    unsigned* err;
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
constexpr unsigned kSiteRows = 0xC0000002u;   // the error word when a request has more than max_q rows, or rows past n_tok,
constexpr unsigned kSiteKeys = 0xC0000003u;   // and when its length passes its row of the table
__device__ __forceinline__ void check_request(const AttnParams& p, int r) {
    if (p.cu && (int64_t) p.cu[r + 1] > min((int64_t) max(p.cu[r], 0) + p.max_q, p.n_tok)) report_error(p.err, kSiteRows);
    if ((int64_t) p.lens[r] > (int64_t) p.width * p.c.bs) report_error(p.err, kSiteKeys);
}
// The first key of row i's window (below zero when it holds all of them).  A row without keys counts as position -1: the
// difference stays in 32 bits for every window.
__device__ __forceinline__ int window_first(const AttnParams& p, const Req& q, int i) { return max(q.len - q.n + i + 1, 0) - p.window; }
// The steps [first, first + n) that the rows of tile rt (of TR rows) see.
template <int TR>
__device__ __forceinline__ void tile_steps(const AttnParams& p, const Req& q, int rt, int& first, int& n) {
    const int rows = q.n * p.G, r0 = rt * TR;
    first = n = 0;
    if (r0 >= rows) return;
    const int i0 = r0 / p.G, i1 = (min(r0 + TR, rows) - 1) / p.G;
    const int hi = q.len - q.n + i1 + 1, lo = p.window > 0 ? max(0, window_first(p, q, i0)) : 0;
    if (hi <= 0) return;
    first = lo / kStep;
    n = (hi + kStep - 1) / kStep - first;
}

// What a step of a tile costs the split, in units: measured per step, a tile of up to 8 rows to one of 9 to 16.
constexpr int kLight = 3, kHeavy = 4;
template <int TR>
__device__ __forceinline__ int step_cost(const AttnParams& p, const Req& q, int rt) {
    return q.n * p.G - rt * TR > 8 ? kHeavy : kLight;
}
__device__ __forceinline__ int64_t units_per_cta(int64_t total, int ctas) {
    return max((int64_t) kAttnWarps * kHeavy, (total + ctas - 1) / ctas);
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Four value codes as fp16 operands, exactly: the byte with its top bit flipped (u = code + 128) under the high byte 0x64
// is the number 1024 + u, and 1152 is subtracted.  Bytes 0, 2 and 1, 3 of a word as two pairs.
__device__ __forceinline__ void code_pairs(uint32_t w, uint32_t& even, uint32_t& odd) {
    constexpr uint32_t mask = 0x00ff00ffu, flip = 0x64806480u;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(even) : "r"(w), "r"(mask), "r"(flip));          // (w & mask) ^ flip
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(odd) : "r"(w >> 8), "r"(mask), "r"(flip));
    const __half2 e = __hsub2(*(const __half2*) &even, *(const __half2*) &flip);
    const __half2 o = __hsub2(*(const __half2*) &odd, *(const __half2*) &flip);
    even = *(const uint32_t*) &e, odd = *(const uint32_t*) &o;
}

// The rows of one tile as right operands for products with the int8 key codes as they are: a row is scaled by a power of
// two to whole numbers of 23 bits, and these are split into signed bytes, most significant first: planes
// [NB][3][D / 32][32 lanes] of 8 bytes.  Sums of int8 products are exact, so the score is that of the scaled query, within
// 2^-23 of the row's largest value a term (two planes, 2^-15, showed in weights of far smaller keys).  rowf[i] undoes the
// scale and holds the score's factor, whose sign the rows carry.  The order of the contraction is the order in which a lane
// reads codes: its 16 consecutive bytes are two depths of 32.
template <int D, int NB>
__device__ __forceinline__ void stage_rows(const AttnParams& p, const Req& q, int h, int rt, uint8_t* qf, float* rowf,
                                           int warp, int n_warps, int lane) {
    const int rows = q.n * p.G;
    constexpr int kPlane = D / 32 * 256, TR = 8 * NB;
    for (int i0 = warp; i0 < TR; i0 += 2 * n_warps) {
        float x[2][D / 32];
#pragma unroll
        for (int k = 0; k < 2; ++k) {                    // two rows' loads at once
            const int i = i0 + k * n_warps, row = rt * TR + i;
            if (i < TR && row < rows) {
                const int64_t at = (int64_t) (q.tok + row / p.G) * p.q_tok + (int64_t) (h * p.G + row % p.G) * p.q_head + lane;
#pragma unroll
                for (int j = 0; j < D / 32; ++j) x[k][j] = load_elem(p.q, at + j * 32, p.type);
            } else {
#pragma unroll
                for (int j = 0; j < D / 32; ++j) x[k][j] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = i0 + k * n_warps;
            if (i >= TR) break;
            float peak = 0.0f;
            bool nan = false;
#pragma unroll
            for (int j = 0; j < D / 32; ++j) peak = fmaxf(peak, fabsf(x[k][j])), nan |= !(fabsf(x[k][j]) <= 3.4028235e38f);
            peak = warp_max(peak);
            nan = __any_sync(0xffffffffu, nan);
            constexpr int top = 148;                     // to [2^21, 2^22): the planes' carries fit
            const int e = min(max((int) (__float_as_uint(peak) >> 23) & 255, 22), 254);
            const float up = copysignf(__uint_as_float((uint32_t) min(127 + top - e, 254) << 23), p.scale_log2);
            const float back = __uint_as_float((uint32_t) max(e - (top - 127), 1) << 23);
            uint8_t* base = qf + (i >> 3) * 3 * kPlane + (i & 7) * 32;
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                // value d of row i: chunk d / 64, quad (d / 16) % 4, byte d % 16 -> depth byte / 8, its place there
                const int d = j * 32 + lane, b = d & 15;
                uint8_t* at = base + ((d >> 6) * 2 + (b >> 3)) * 256 + ((d >> 4) & 3) * 8 + (b & 7);
                int v = __float2int_rn(x[k][j] * up);
#pragma unroll
                for (int l = 2; l >= 0; --l) {
                    at[l * kPlane] = (uint8_t) v;
                    v = (v - (int) (int8_t) v) >> 8;
                }
            }
            if (lane == 0) rowf[i] = nan ? __uint_as_float(0x7fffffffu) : fabsf(p.scale_log2) * back;   // NaN or infinity: a NaN row
        }
    }
}

// A warp's running rows, NB groups of 8.  Lane (g, quad) holds rows 2 quad and 2 quad + 1 of a group and the output columns
// whose codes it reads: tile j of 16 columns of the transposed product is the bytes 2 j, 2 j + 1 of every lane's piece.
template <int D, int NB>
struct Rows {
    float4 o[NB][D / 16];            // {column 2 j: row 2 quad, row + 1; column 2 j + 1: row 2 quad, row + 1}
    float m[NB][2], l[NB][2];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int u = 0; u < NB; ++u) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) o[u][i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            m[u][0] = m[u][1] = -INFINITY;
            l[u][0] = l[u][1] = 0.0f;
        }
    }
    // the first of 2 * (tiles) consecutive columns that tiles j, j + 1, .. hold
    __device__ static __forceinline__ int column(int j, int g) { return D == 64 ? g * 8 + 2 * j : (j / 8) * 128 + g * 16 + 2 * (j % 8); }
};

constexpr float kShift = 15.0f;  // weights are exp2(x - the row's largest so far + 15): at most 2^15, and fp16 keeps 11 bits
                                 // of those down to 2^-29 of the largest

// A warp's ring of steps in shared memory: per step 16 tokens' key codes and their value codes, 16-byte pieces permuted so
// that a quarter warp's reads touch every bank once, and {key scale, value scale, whether the block is in the cache}.
// Depths by what fits the CTAs a SM holds: 80 to 130 KB a SM are in flight.
//   head_dim 128, 256: piece ^ (2 ((row / 2) % 4) ^ 4 (row % 2)) within its 128 bytes
//   head_dim 64: keys as they are; value rows in the order 0 2 4 6 1 3 5 7 (and + 8), piece ^ 2 (their place / 2 % 2)
template <int D>
struct Ring {
    static constexpr int kDepth = D == 256 ? 2 : D == 128 ? 3 : 5;
    static constexpr int kHalf = kStep * D;
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kHeads = kDepth * kStage;
    static constexpr int kBytes = kHeads + 128;
    static constexpr int kRow1 = D == 64 ? 4 * D : D;      // from a lane's even value row to the odd one, before the xor
    // byte offsets of 16-byte piece `lane` of a step (piece 32 i + lane: xor the rows' change, plus 512 i) ...
    __device__ static __forceinline__ int put_k(int lane) {
        const int row = lane / (D / 16), piece = lane % (D / 16);
        return D == 64 ? lane * 16 : row * D + ((piece ^ swizzle(row)) << 4);
    }
    __device__ static __forceinline__ int put_v(int lane) {
        if (D != 64) return put_k(lane);
        const int row = lane >> 2, piece = lane & 3, at = ((row & 1) << 2) | (row >> 1);
        return at * D + ((piece ^ (((at >> 1) & 1) << 1)) << 4);
    }
    // ... and of what lane (g, quad) reads: key row g, piece quad; value row 2 quad, piece g (D 64: half a piece)
    __device__ static __forceinline__ int get_k(int g, int qd) {
        return D == 64 ? g * D + qd * 16 : g * D + ((qd ^ swizzle(g)) << 4);
    }
    __device__ static __forceinline__ int get_v(int g, int qd) {
        return D == 64 ? qd * D + (((g >> 1) ^ (((qd >> 1) & 1) << 1)) << 4) + (g & 1) * 8
                       : 2 * qd * D + ((g ^ swizzle(2 * qd)) << 4);
    }
    __device__ static __forceinline__ int swizzle(int row) { return (((row >> 1) & 3) << 1) ^ ((row & 1) << 2); }
};
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// A warp's walk over steps first + off, first + off + stride, ... below first + n of request r's keys and values, for one
// tile of rows.  The constructor begins the copies (the rows need not be staged yet), run() does the rest.
// Both products are transposed, keys and value columns as the 16 rows of the instruction and queries as its 8 columns: a
// decode step has at most 8 rows a head in most models, and a tile of queries by 16 would be half empty, at twice the
// products, registers and exponentials.  x = q . k (int8 products, exact) times the block's key scale and the row's; the
// online softmax's largest score m and sum l in fp32 (the lanes compare their scores with m; only when one is larger do
// they meet); o += weights . codes times the block's value scale.
// SP 1, bf16 outputs: weights, times 2^15 and the value scale relative to the largest so far, enter the product as one
//   fp16 value (11 bits down to 2^-29 of the largest weight; 2^-40 of it below) and o accumulates in the tensor cores.
// SP 2, fp32 and fp16 outputs: weights as two fp16 values; a step's product starts from zero and is added in fp32 times the value
//   scale, since the tensor cores' sums truncate.
template <int D, int SP>
struct Walk {
    const AttnParams& p;
    const int32_t* tab;
    uint32_t ring, put_k, put_v;
    int shift, first, n, stride, h, lane;
    int s, s_copy, stage_copy, id_copy;

    __device__ __forceinline__ Walk(const AttnParams& p, uint32_t ring, int r, int h, int first, int n, int off, int stride, int lane)
        : p(p), tab(p.table + (int64_t) r * p.table_stride), ring(ring), put_k(Ring<D>::put_k(lane)),
          put_v(Ring<D>::kHalf + Ring<D>::put_v(lane)), shift(p.c.bs >> 6 ? 2 : p.c.bs >> 5), first(first), n(n), stride(stride), h(h),
          lane(lane), s(off), s_copy(off), stage_copy(0) {
        id_copy = block(s_copy);
#pragma unroll
        for (int i = 0; i < Ring<D>::kDepth - 1; ++i) copy();
    }
    __device__ __forceinline__ int block(int x) const { return x < n ? __ldg(tab + ((first + x) >> shift)) : 0; }
    // the next step's codes and scales on their way (one group, empty past the last step)
    __device__ __forceinline__ void copy() {
        if (s_copy < n) {
            const bool ok = id_copy >= 0 && id_copy < p.c.n_blocks;
            const int64_t bh = (int64_t) (ok ? id_copy : 0) * p.c.H + h;
            const int64_t at = (bh * p.c.bs + (((first + s_copy) & ((1 << shift) - 1)) * kStep)) * D + lane * 16;
            const uint32_t dst = ring + stage_copy * Ring<D>::kStage, head = ring + Ring<D>::kHeads + stage_copy * 16;
            const uint32_t k0 = dst + put_k, v0 = dst + put_v;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const uint32_t x = D == 256 ? 32 * (i & 3) : D == 128 ? 64 * (i & 1) : 0;
                cp_async16((k0 ^ x) + i * 512, p.c.k + at + i * 512);
                cp_async16((v0 ^ x) + i * 512, p.c.v + at + i * 512);
            }
            if (lane == 0) cp4(head, p.c.ks + bh);
            if (lane == 1) cp4(head + 4, p.c.vs + bh);
            if (lane == 2) asm volatile("st.shared.u32 [%0], %1;" ::"r"(head + 8), "r"((int) ok) : "memory");
        }
        cp_commit();
        s_copy += stride;
        id_copy = block(s_copy);
        stage_copy = stage_copy + 1 == Ring<D>::kDepth ? 0 : stage_copy + 1;
    }

    // tile rt of TR rows, its first NB groups
    template <int TR, int NB, int NBR>
    __device__ __forceinline__ void run(const Req& q, int rt, const uint8_t* qf, const float* rowf, Rows<D, NBR>& R) {
        const int g = lane >> 2, qd = lane & 3, rows = q.n * p.G;
        constexpr bool QREG = NB == 1 && D <= 128;       // the rows' operands stay in registers where they fit
        const uint2* qp = (const uint2*) qf + lane;
        uint2 qr[QREG ? 3 * D / 32 : 1];
        if constexpr (QREG) {
#pragma unroll
            for (int i = 0; i < 3 * D / 32; ++i) qr[i] = qp[i * 32];
        }
        const uint32_t get_k = Ring<D>::get_k(g, qd), get_v = Ring<D>::kHalf + Ring<D>::get_v(g, qd);
        int pos[NB][2];                                  // a row sees the keys up to pos, the last `window` of them
        float rf[NB][2];
#pragma unroll
        for (int u = 0; u < NB; ++u)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                pos[u][i] = q.len - q.n + min(rt * TR + u * 8 + 2 * qd + i, rows - 1) / p.G;
                rf[u][i] = rowf[u * 8 + 2 * qd + i];
            }
        const int pmin = q.len - q.n + (rt * TR) / p.G;
        const int lmax = p.window > 0 ? window_first(p, q, (min(rt * TR + TR, rows) - 1) / p.G) : INT_MIN;
        float ref = 0.0f, per_ref = 0.0f;                // SP 1: a power of two above the value scales so far, its inverse
        int stage = 0;
        for (; s < n; s += stride) {
            __syncwarp();                                // the stage that copy() fills is read
            copy();
            cp_wait<Ring<D>::kDepth - 1>();
            __syncwarp();
            const uint32_t at = ring + stage * Ring<D>::kStage;
            const uint4 head = lds16(ring + Ring<D>::kHeads + stage * 16);
            stage = stage + 1 == Ring<D>::kDepth ? 0 : stage + 1;
            if (head.z == 0) continue;                   // a block outside the cache
            const float ks = __uint_as_float(head.x), vs = __uint_as_float(head.y);

            int xi[NB][3][4];
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const uint32_t ka = ((at + get_k) ^ ((i & 1) * 64)) + (i >> 1) * 128;
                const uint4 k0 = lds16(ka), k1 = lds16(ka + 8 * D);
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    const uint32_t a[4] = {word(k0, 2 * kk), word(k1, 2 * kk), word(k0, 2 * kk + 1), word(k1, 2 * kk + 1)};
#pragma unroll
                    for (int u = 0; u < NB; ++u)
#pragma unroll
                        for (int l = 0; l < 3; ++l) {
                            const uint2 b = QREG ? qr[QREG ? l * (D / 32) + i * 2 + kk : 0] : qp[(u * 3 * (D / 32) + l * (D / 32) + i * 2 + kk) * 32];
                            if (i == 0 && kk == 0) mma_s8_zero(xi[u][l], a, b.x, b.y);
                            else mma_s8(xi[u][l], a, b.x, b.y);
                        }
                }
            }
            // y[e]: token g + 8 (e / 2), row 2 quad + e % 2
            float y[NB][4], sc[NB][2];
            const int t0 = (first + s) * kStep;
            const bool edge = t0 + kStep - 1 > pmin || t0 < lmax;
            bool moved = SP == 1 && vs > ref;
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                sc[u][0] = ks * rf[u][0], sc[u][1] = ks * rf[u][1];
#pragma unroll
                for (int e = 0; e < 4; ++e) y[u][e] = fmaf((float) xi[u][0][e], 65536.0f, (float) (xi[u][1][e] * 256 + xi[u][2][e])) * sc[u][e & 1];
                if (edge) {
                    const int w = p.window > 0 ? p.window : INT_MAX;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int t = t0 + g + 8 * (e >> 1);
                        if (t > pos[u][e & 1] || pos[u][e & 1] - t >= w) y[u][e] = -INFINITY;
                    }
                }
                moved |= fmaxf(y[u][0], y[u][2]) > R.m[u][0] || fmaxf(y[u][1], y[u][3]) > R.m[u][1];
            }
            if (__any_sync(0xffffffffu, moved)) {
                float by = 1.0f;
                if (SP == 1 && vs > ref) {
                    const uint32_t e = max(min((__float_as_uint(vs) >> 23) + 1, 253u), 2u);      // 2^(e - 127) > vs
                    by = ref * __uint_as_float((254 - e) << 23);
                    ref = __uint_as_float(e << 23), per_ref = __uint_as_float((254 - e) << 23);
                }
#pragma unroll
                for (int u = 0; u < NB; ++u) {
                    float al[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float mx = fmaxf(R.m[u][i], fmaxf(y[u][i], y[u][2 + i]));
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        al[i] = mx == -INFINITY ? 1.0f : ex2(R.m[u][i] - mx);
                        R.m[u][i] = mx;
                        R.l[u][i] *= al[i];
                        al[i] *= by;
                    }
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        R.o[u][j].x *= al[0], R.o[u][j].y *= al[1], R.o[u][j].z *= al[0], R.o[u][j].w *= al[1];
                    }
                }
            }
            uint32_t b[NB][2], bl[NB][2];
            const float r = SP == 1 ? vs * per_ref : 1.0f;
#pragma unroll
            for (int u = 0; u < NB; ++u) {
                const float z[2] = {R.m[u][0] == -INFINITY ? 0.0f : kShift - R.m[u][0], R.m[u][1] == -INFINITY ? 0.0f : kShift - R.m[u][1]};
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = ex2(y[u][e] + z[e & 1]);
                R.l[u][0] += w[0] + w[2], R.l[u][1] += w[1] + w[3];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t hi = pack_f16(w[2 * e] * r, w[2 * e + 1] * r);
                    b[u][e] = transpose8(hi);
                    if (SP == 2) {
                        const float2 f = __half22float2(*(const __half2*) &hi);
                        bl[u][e] = transpose8(pack_f16(w[2 * e] - f.x, w[2 * e + 1] - f.y));
                    }
                }
            }
            const uint32_t va = at + get_v, vb = D == 64 ? va + Ring<D>::kRow1 : (va ^ 64) + Ring<D>::kRow1;
#pragma unroll
            for (int i = 0; i < (D + 127) / 128; ++i) {
                uint4 v[4];                              // tokens 2 quad, 2 quad + 1, 2 quad + 8, 2 quad + 9
                if constexpr (D == 64) {
                    const uint2 a = lds8(va), c = lds8(vb), d = lds8(va + 8 * D), e = lds8(vb + 8 * D);
                    v[0] = make_uint4(a.x, a.y, 0, 0), v[1] = make_uint4(c.x, c.y, 0, 0);
                    v[2] = make_uint4(d.x, d.y, 0, 0), v[3] = make_uint4(e.x, e.y, 0, 0);
                } else {
                    v[0] = lds16(va + i * 128), v[1] = lds16(vb + i * 128);
                    v[2] = lds16(va + i * 128 + 8 * D), v[3] = lds16(vb + i * 128 + 8 * D);
                }
#pragma unroll
                for (int w = 0; w < (D == 64 ? 2 : 4); ++w) {
                    uint32_t c0[4], c1[4];               // bytes 0 .. 3 of the word: two tokens side by side, and eight on
                    code_pairs(__byte_perm(word(v[0], w), word(v[1], w), 0x6420), c0[0], c0[2]);
                    code_pairs(__byte_perm(word(v[0], w), word(v[1], w), 0x7531), c0[1], c0[3]);
                    code_pairs(__byte_perm(word(v[2], w), word(v[3], w), 0x6420), c1[0], c1[2]);
                    code_pairs(__byte_perm(word(v[2], w), word(v[3], w), 0x7531), c1[1], c1[3]);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t a[4] = {c0[2 * j], c0[2 * j + 1], c1[2 * j], c1[2 * j + 1]};
#pragma unroll
                        for (int u = 0; u < NB; ++u) {
                            float4& o = R.o[u][i * 8 + w * 2 + j];
                            if constexpr (SP == 1) {
                                mma_f16(o, a, b[u][0], b[u][1]);
                            } else {
                                float acc[4];
                                mma_f16_zero(acc, a, b[u][0], b[u][1]);
                                mma_f16(acc, a, bl[u][0], bl[u][1]);
                                o.x = fmaf(vs, acc[0], o.x), o.y = fmaf(vs, acc[1], o.y);
                                o.z = fmaf(vs, acc[2], o.z), o.w = fmaf(vs, acc[3], o.w);
                            }
                        }
                    }
                }
            }
        }
        cp_wait<0>();                                    // (only empty groups are left)
#pragma unroll
        for (int u = 0; u < NB; ++u) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {                // the lanes of a column hold parts of its row's sum
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) R.l[u][i] += __shfl_xor_sync(0xffffffffu, R.l[u][i], o);
            }
            if (SP == 1) {
#pragma unroll
                for (int j = 0; j < D / 16; ++j) R.o[u][j].x *= ref, R.o[u][j].y *= ref, R.o[u][j].z *= ref, R.o[u][j].w *= ref;
            }
        }
    }
};

// N values (2 at D 64, else a multiple of 4) to consecutive elements; `wide`: N elements are one aligned access.
template <int N>
__device__ __forceinline__ void store_row(void* o, int64_t at, int type, const float (&x)[N], bool wide) {
    if (!wide) {
#pragma unroll
        for (int i = 0; i < N; ++i) store_elem(o, at + i, type, x[i]);
    } else if (type == E_F32) {
#pragma unroll
        for (int i = 0; i < N; i += 2) *(float2*) ((float*) o + at + i) = make_float2(x[i], x[i + 1]);
    } else {
        uint32_t u[N / 2];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) u[i] = type == E_F16 ? pack_f16(x[2 * i], x[2 * i + 1]) : pack_bf16(x[2 * i], x[2 * i + 1]);
        if constexpr (N >= 8) {
#pragma unroll
            for (int i = 0; i < N / 8; ++i) *((uint4*) ((uint16_t*) o + at) + i) = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
        } else if constexpr (N == 4) {
            *(uint2*) ((uint16_t*) o + at) = make_uint2(u[0], u[1]);
        } else {
            *(uint32_t*) ((uint16_t*) o + at) = u[0];
        }
    }
}

// CTAs a SM holds, for tiles of 8 (NB 1) and of 16 rows (NB 2, where a request has more than 8: a step's codes are then
// read and turned into operands once for both groups; tiles with up to 8 rows skip the second)
template <int D, int NB>
constexpr int kSplitCtas = NB == 1 ? (D == 256 ? 3 : D == 128 ? 4 : 5) : (D == 256 ? 2 : D == 128 ? 3 : 4);

// The steps of all (request, head, tile) segments, one after the other (request, then head, then tile), are cut into
// equal ranges, one per CTA; a range's warps take its steps in turn and join their rows through shared memory at the
// end of each segment.  A segment inside one range is finished there; one cut by a range's end leaves its rows, maxima
// and sums for k_attn_join.  So a lone request of 131,072 tokens and 64 requests of uneven lengths fill the GPU alike.
// Bound by memory with one query a request (32 requests of 8192 tokens, heads of 128: 5.7 TB/s; 2 of 131,072, heads of 256,
// fp32: 59 us, 4.6 TB/s), by latency with more (64 of up to 8192 with up to 3: 139 us, 4.0 TB/s): the two groups' rows leave
// 12 warps a SM (168 registers), issue slots are 53% active, and the chain of products, maxima and weights is what a warp
// waits for (1.6 cycles an instruction), not a pipe.
template <int D, int SP, int NB>
__global__ void __launch_bounds__(kAttnWarps * 32, kSplitCtas<D, NB>) k_attn_split(const __grid_constant__ AttnParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* rings = smem;                                             // [warps] rings; then [warps][8 NB][D] rows to join
    constexpr int TR = 8 * NB;
    float4* mrg = (float4*) rings;
    uint8_t* qf = rings + kAttnWarps * Ring<D>::kBytes;                // [NB][3][D / 32][32][8]
    float* ml = (float*) (qf + NB * 3 * (D / 32) * 256);               // [warps][2][TR]
    float* rowf = ml + kAttnWarps * 2 * TR;                            // [TR]
    int64_t* pre = (int64_t*) (rowf + TR);                             // [n_req + 1]
    static_assert(Ring<D>::kBytes >= TR * D * 4, "the rows to join lie over the rings");
    __shared__ int64_t wsum[kAttnWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int R = p.n_req, T = kAttnWarps * 32;
    // units before each request
    {
        const int per = (R + T - 1) / T, r0 = min(tid * per, R), r1 = min(r0 + per, R);
        int64_t sum = 0;
        for (int r = r0; r < r1; ++r) {
            const Req q = attn_req(p, r);
            for (int rt = 0; rt < p.tiles; ++rt) {
                int f, n;
                tile_steps<TR>(p, q, rt, f, n);
                sum += (int64_t) n * p.c.H * step_cost<TR>(p, q, rt);
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
        if (per == 1) {
            if (r0 < r1) pre[r0] = x;
            x += sum;
        } else {
            for (int r = r0; r < r1; ++r) {
                pre[r] = x;
                const Req q = attn_req(p, r);
                for (int rt = 0; rt < p.tiles; ++rt) {
                    int f, n;
                    tile_steps<TR>(p, q, rt, f, n);
                    x += (int64_t) n * p.c.H * step_cost<TR>(p, q, rt);
                }
            }
        }
        if (tid == T - 1) pre[R] = x;
        __syncthreads();
    }
    if (blockIdx.x == 0)
        for (int r = tid; r <= R; r += T) p.pre[r] = pre[r];
    asm volatile("griddepcontrol.launch_dependents;");
    const int64_t total = pre[R];
    const int64_t per_cta = units_per_cta(total, gridDim.x);
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
        const int64_t all = (pre[r + 1] - pre[r]) / p.c.H;        // units of one head
        const int h = (int) ((at - pre[r]) / all);
        int64_t in = (at - pre[r]) - (int64_t) h * all;
        int rt = 0, first = 0, n = 0, cost = kLight;
        for (;; ++rt) {
            tile_steps<TR>(p, q, rt, first, n);
            cost = step_cost<TR>(p, q, rt);
            if (in < (int64_t) n * cost) break;
            in -= (int64_t) n * cost;
        }
        const int64_t seg = at - in;                              // where the segment starts
        const int64_t stop = min((int64_t) n * cost, end - seg);
        at = seg + stop;
        const int s0 = (int) ((in + cost - 1) / cost), take = (int) ((stop + cost - 1) / cost) - s0;
        if (take <= 0) continue;                                  // the range ends within a step: the next one's
        Walk<D, SP> walk(p, smem_u32(rings + warp * Ring<D>::kBytes), r, h, first + s0, take, warp, kAttnWarps, lane);
        stage_rows<D, NB>(p, q, h, rt, qf, rowf, warp, kAttnWarps, lane);
        __syncthreads();
        Rows<D, NB> rows;
        rows.clear();
        const int n_rows = q.n * p.G;
        if (NB == 1 || n_rows - rt * TR > 8) walk.template run<TR, NB>(q, rt, qf, rowf, rows);
        else walk.template run<TR, 1>(q, rt, qf, rowf, rows);
        const int g = lane >> 2, qd = lane & 3;
        __syncthreads();                                          // the rings are free
#pragma unroll
        for (int u = 0; u < NB; ++u) {
#pragma unroll
            for (int j = 0; j < D / 16; ++j) mrg[((warp * NB + u) * (D / 16) + j) * 32 + lane] = rows.o[u][j];
            if (g == 0) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    ml[warp * 2 * TR + u * 8 + 2 * qd + i] = rows.m[u][i];
                    ml[warp * 2 * TR + TR + u * 8 + 2 * qd + i] = rows.l[u][i];
                }
            }
        }
        __syncthreads();
        // warp w joins the four warps' tiles w D / 64 .. (w + 1) D / 64
        constexpr int JT = D / 16 / kAttnWarps;
        const int64_t slot = 2 * (int64_t) blockIdx.x + (seg > begin ? 1 : 0);
        const int col = Rows<D, NB>::column(warp * JT, g);
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            if (rt * TR + u * 8 >= n_rows) continue;
            float m[2], l[2] = {0.0f, 0.0f}, f[2][kAttnWarps], x[2][2 * JT];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float* st = ml + u * 8 + 2 * qd + i;
                m[i] = -INFINITY;
#pragma unroll
                for (int w = 0; w < kAttnWarps; ++w) m[i] = fmaxf(m[i], st[w * 2 * TR]);
#pragma unroll
                for (int w = 0; w < kAttnWarps; ++w) {
                    const float mw = st[w * 2 * TR];
                    f[i][w] = mw == -INFINITY ? 0.0f : ex2(mw - m[i]);
                    l[i] = fmaf(st[w * 2 * TR + TR], f[i][w], l[i]);
                }
            }
#pragma unroll
            for (int j = 0; j < JT; ++j) {
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kAttnWarps; ++w) {
                    const float4 v = mrg[((w * NB + u) * (D / 16) + warp * JT + j) * 32 + lane];
                    o.x = fmaf(v.x, f[0][w], o.x), o.y = fmaf(v.y, f[1][w], o.y);
                    o.z = fmaf(v.z, f[0][w], o.z), o.w = fmaf(v.w, f[1][w], o.w);
                }
                x[0][2 * j] = o.x, x[1][2 * j] = o.y, x[0][2 * j + 1] = o.z, x[1][2 * j + 1] = o.w;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int row = u * 8 + 2 * qd + i, all_row = rt * TR + row;
                if (all_row >= n_rows) continue;
                if (take == n) {
                    const float inv = l[i] > 0.0f ? 1.0f / l[i] : 0.0f;     // a row that sees no key is zero
                    const int64_t to = (int64_t) (q.tok + all_row / p.G) * p.o_tok + (int64_t) (h * p.G + all_row % p.G) * p.o_head;
#pragma unroll
                    for (int j = 0; j < 2 * JT; ++j) x[i][j] *= inv;
                    store_row<2 * JT>(p.o, to + col, p.type, x[i], p.wide_out);
                } else {
                    float* to = p.part + (slot * TR + row) * D + col;
#pragma unroll
                    for (int j = 0; j < 2 * JT; j += 2) *(float2*) (to + j) = make_float2(x[i][j], x[i][j + 1]);
                    if (warp == 0 && g == 0) {
                        float* st = p.part + 2 * (int64_t) p.n_cta * TR * D + slot * 2 * TR;
                        st[row] = m[i], st[TR + row] = l[i];
                    }
                }
            }
        }
        __syncthreads();                                          // the rows are joined
    }
}

// CTA (segment, share): the parts of the rows of a segment that was cut, joined by their maxima, row and 64 columns at a time:
// a warp an item when the parts are few, all eight warps on one item, parts in turn, when they are many (a long request).
// Zeros for the rows of a segment without keys.  Segments inside one range were finished by k_attn_split.  What the parts
// do not decide is read before the wait for the split's end.
template <int D, int TR>
__global__ void __launch_bounds__(256) k_attn_join(const __grid_constant__ AttnParams p) {
    __shared__ float2 acc[8][32];
    __shared__ float stat[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int seg_id = blockIdx.x;
    if (seg_id == (int) gridDim.x - 1) {                     // past the segments: the requests' bounds
        if (blockIdx.y == 0)
            for (int i = threadIdx.x; i < p.n_req; i += 256) check_request(p, i);
        return;
    }
    const int rt = seg_id % p.tiles, h = seg_id / p.tiles % p.c.H, r = seg_id / p.tiles / p.c.H;
    const Req q = attn_req(p, r);
    int first, n;
    int64_t seg = 0;
    for (int t = 0; t < rt; ++t) {
        tile_steps<TR>(p, q, t, first, n);
        seg += (int64_t) n * step_cost<TR>(p, q, t);
    }
    tile_steps<TR>(p, q, rt, first, n);
    const int cost = step_cost<TR>(p, q, rt);
    const int items = min(max(q.n * p.G - rt * TR, 0), TR) * (D / 64);
    asm volatile("griddepcontrol.wait;" ::: "memory");       // every CTA: the split is complete from here on
    if (items == 0) return;
    const int64_t total = p.pre[p.n_req], p0 = p.pre[r], p1 = p.pre[r + 1], per_cta = units_per_cta(total, p.n_cta);
    seg += p0 + (p1 - p0) / p.c.H * h;
    const int c0 = (int) (seg / per_cta);
    int c1 = n ? (int) ((seg + (int64_t) n * cost - 1) / per_cta) : c0;
    if (n) {
        if (((c0 + 1) * per_cta - seg + cost - 1) / cost >= n) return;                    // finished by the split
        if ((c1 * per_cta - seg + cost - 1) / cost >= n) --c1;                            // its share was within a step
    }
    const float* stats = p.part + 2 * (int64_t) p.n_cta * TR * D;
    auto slot = [&](int c) { return 2 * c + (seg > c * per_cta ? 1 : 0); };
    auto join = [&](int i, int col, int from, int by, float2& a, float& l) {
        float m = -INFINITY;
        for (int c = c0 + lane; c <= c1; c += 32) m = fmaxf(m, stats[slot(c) * 2 * TR + i]);
        m = warp_max(m);
        a = make_float2(0.0f, 0.0f), l = 0.0f;
#pragma unroll 8
        for (int c = c0 + from; c <= c1; c += by) {
            const int sl = slot(c);
            const float mc = stats[sl * 2 * TR + i], lc = stats[sl * 2 * TR + TR + i];
            const float2 b = *(const float2*) (p.part + ((int64_t) sl * TR + i) * D + col);
            const float f = mc == -INFINITY ? 0.0f : ex2(mc - m);
            l = fmaf(lc, f, l);
            a.x = fmaf(b.x, f, a.x), a.y = fmaf(b.y, f, a.y);
        }
    };
    auto write = [&](int i, int col, float2 a, float l) {
        const int row = rt * TR + i;
        const int64_t out = (int64_t) (q.tok + row / p.G) * p.o_tok + (int64_t) (h * p.G + row % p.G) * p.o_head + col;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        const float x[2] = {a.x * inv, a.y * inv};
        store_row<2>(p.o, out, p.type, x, p.wide_out);
    };
    if (n == 0 || c1 - c0 < 16) {
        for (int it = blockIdx.y * 8 + warp; it < items; it += gridDim.y * 8) {
            const int i = it / (D / 64), col = it % (D / 64) * 64 + 2 * lane;
            float2 a = make_float2(0.0f, 0.0f);
            float l = 0.0f;
            if (n) join(i, col, 0, 1, a, l);
            write(i, col, a, l);
        }
        return;
    }
    for (int it = blockIdx.y; it < items; it += gridDim.y) {
        const int i = it / (D / 64), col = it % (D / 64) * 64 + 2 * lane;
        float2 a;
        float l;
        join(i, col, warp, 8, a, l);
        acc[warp][lane] = a;
        if (lane == 0) stat[warp] = l;
        __syncthreads();
        if (warp == 0) {
            l = 0.0f;
            a = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < 8; ++w) l += stat[w], a.x += acc[w][lane].x, a.y += acc[w][lane].y;
            write(i, col, a, l);
        }
        __syncthreads();
    }
}

// check_request for k_attn_tiles, whose registers are so full that the same lines inside it cost 4 to 7% (843 queries over 2000
// keys: 281 to 290 us against 271 without and 276 with this launch).
__global__ void __launch_bounds__(256) k_attn_check(const __grid_constant__ AttnParams p) {
    asm volatile("griddepcontrol.launch_dependents;");
    for (int r = threadIdx.x; r < p.n_req; r += 256) check_request(p, r);
}

// Many rows of fp32 queries: one warp per tile of 32 rows (head_dim 256: 16), every step of the tile by the same warp, which turns a
// step's codes into operands once for all of them; the four warps of a CTA take neighbouring tiles of a head, so they share
// the codes through the caches.  Bound by the latency of a step's products and weights at 8 warps a SM (255 registers; issue
// slots 41% active): 843 queries of 32 heads over 8, 2000 keys, heads of 128, 271 us, 80 TFLOP/s; of 8 heads over one, which are
// 53 CTAs, 209.
template <int D>
constexpr int kTileGroups = D == 256 ? 2 : 4;
template <int D>
__global__ void __launch_bounds__(kAttnWarps * 32) k_attn_tiles(const __grid_constant__ AttnParams p) {
    constexpr int NB = kTileGroups<D>, TR = 8 * NB;
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int kQ = NB * 3 * (D / 32) * 256;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint8_t* ring = smem + warp * (Ring<D>::kBytes + kQ + 128);
    uint8_t* qf = ring + Ring<D>::kBytes;
    float* rowf = (float*) (qf + kQ);
    const int rt = (gridDim.x - 1 - blockIdx.x) * kAttnWarps + warp, h = blockIdx.y, r = blockIdx.z;
    const Req q = attn_req(p, r);
    if (rt * TR >= q.n * p.G) return;
    int first, n;
    tile_steps<TR>(p, q, rt, first, n);
    Walk<D, 2> walk(p, smem_u32(ring), r, h, first, n, 0, 1, lane);
    stage_rows<D, NB>(p, q, h, rt, qf, rowf, 0, 1, lane);
    __syncwarp();
    Rows<D, NB> rows;
    rows.clear();
    walk.template run<TR, NB>(q, rt, qf, rowf, rows);
    const int g = lane >> 2, qd = lane & 3, n_rows = q.n * p.G;
#pragma unroll
    for (int u = 0; u < NB; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = rt * TR + u * 8 + 2 * qd + i;
            if (row >= n_rows) continue;
            const float inv = rows.l[u][i] > 0.0f ? 1.0f / rows.l[u][i] : 0.0f;
            const int64_t to = (int64_t) (q.tok + row / p.G) * p.o_tok + (int64_t) (h * p.G + row % p.G) * p.o_head;
#pragma unroll
            for (int j0 = 0; j0 < D / 16; j0 += 4) {
                float x[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 o = rows.o[u][j0 + j];
                    x[2 * j] = (i ? o.y : o.x) * inv, x[2 * j + 1] = (i ? o.w : o.z) * inv;
                }
                store_row<8>(p.o, to + Rows<D, NB>::column(j0, g), p.type, x, p.wide_out);
            }
        }
}

}  // namespace
}  // namespace tsb
#include "tsb_cache_prompt.cuh"
namespace tsb {
unsigned* device_error_word();          // tsb_moe.cu: the current device's error word
namespace {

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
    return Cache{c->k, c->v, c->k_scale, c->v_scale, c->n_blocks, c->block_size, c->n_kv_heads, c->head_dim,
                 c->block_size == 16 ? 4 : c->block_size == 32 ? 5 : 6};
}
bool elem_ok(int t) { return t == E_F32 || t == E_F16 || t == E_BF16; }

struct AttnPlan {
    int G, tiles, n_cta, groups;
    bool split, prompt;
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
    // (k_attn_prompt looks up the blocks of up to three tiles of 128 tokens past a request's last in 32 bits)
    if ((int64_t) d->table_width * c->block_size > 0x7fffffffll - 1024 || c->n_kv_heads > 65535)
        return cfail(TSB_ERR_UNSUPPORTED, "kv8_attention: at most 2^31 - 1025 tokens a request and 65535 heads");
    a.G = d->q_heads / c->n_kv_heads;
    const int64_t rows = (int64_t) d->max_q * a.G;
    if (rows > (1 << 28)) return cfail(TSB_ERR_UNSUPPORTED, "kv8_attention: too many query rows");
    // Rows a key / value head has (queries x heads of its group).  Up to 64 the steps of a request are split over CTAs; above,
    // tiles of rows walk all of their keys, 16-bit queries in tiles of 128 on tcgen05.  More rows are split too while their
    // tiles would leave most SMs idle.  Measured, split against tiles (us): 64 rows, 16 requests of 2000 keys, 41 against 49
    // (fp32 43 against 212); 128 rows of them 60 against 54; 512 rows in 8 tiles, 3000 keys of 256, 58 against 102; 768 rows in
    // 12 tiles, 2000 keys, 54 against 54; 512 rows in 16, 128 keys, 40 against 23.  The fp32 tiles are smaller and slower:
    // 1536 rows in 24 tiles, 3000 keys, 101 against 303; 4096 in 32, 2000 keys, 174 against 210; 6744 in 53 293 against 209.
    const int64_t prompt_ctas = (rows + 127) / 128 * c->n_kv_heads * d->n_req;
    a.split = rows <= kSplitRows || prompt_ctas < (d->elem_type == E_F32 ? kPromptCtas32 : kPromptCtas);
    a.prompt = !a.split && d->elem_type != E_F32;
    a.groups = a.prompt ? 16 : !a.split ? (c->head_dim == 256 ? kTileGroups<256> : kTileGroups<128>) : rows <= 8 ? 1 : 2;
    a.tiles = (int) ((rows + 8 * a.groups - 1) / (8 * a.groups));
    const int sms = sm_count();
    if (!sms) return cfail(TSB_ERR_CUDA, "kv8_attention: no CUDA device");
    const int d_ = c->head_dim;
    a.n_cta = sms * (a.groups == 1 ? (d_ == 256 ? kSplitCtas<256, 1> : d_ == 128 ? kSplitCtas<128, 1> : kSplitCtas<64, 1>)
                                   : (d_ == 256 ? kSplitCtas<256, 2> : d_ == 128 ? kSplitCtas<128, 2> : kSplitCtas<64, 2>));
    a.ws = a.split ? (((uint64_t) d->n_req + 1) * 8 + 255) / 256 * 256 + (uint64_t) a.n_cta * 2 * 8 * a.groups * (c->head_dim + 2) * 4 : 0;
    return TSB_OK;
}

template <int D, int SP, int NB>
int launch_split(const AttnParams& p, const AttnPlan& a, int rows, cudaStream_t st) {
    static std::atomic<bool> granted[kMaxDev];
    constexpr int fixed = kAttnWarps * Ring<D>::kBytes + NB * (3 * (D / 32) * 256 + kAttnWarps * 64 + 32);
    const int sm = fixed + (p.n_req + 1) * 8;
    if (int rc = allow_smem(k_attn_split<D, SP, NB>, granted, fixed + (kMaxReq + 1) * 8, "kv8_attention: shared memory")) return rc;
    k_attn_split<D, SP, NB><<<a.n_cta, kAttnWarps * 32, sm, st>>>(p);
    if (int rc = ccuda("kv8_attention")) return rc;
    // the join's CTAs come up while the split runs; each waits for it (griddepcontrol.wait) before it reads its results
    cudaLaunchConfig_t cfg{};
    const int segs = p.n_req * p.c.H * p.tiles, items = std::min(rows, 8 * NB) * (D / 64);
    cfg.gridDim = dim3((unsigned) segs + 1, (unsigned) std::max(1, std::min(items, a.n_cta / segs)));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, k_attn_join<D, 8 * NB>, p);
    return ccuda("kv8_attention: join");
}
template <int D, bool LO>
int launch_prompt(const AttnParams& p, cudaStream_t st) {
    static std::atomic<bool> granted[kMaxDev];
    if (int rc = allow_smem(k_attn_prompt<D, LO>, granted, Prompt<D, LO>::kAsk, "kv8_attention: shared memory")) return rc;
    k_attn_prompt<D, LO><<<dim3((unsigned) p.tiles, p.c.H, p.n_req), kPromptThreads, Prompt<D, LO>::kAsk, st>>>(p);
    return ccuda("kv8_attention");
}
template <int D, int SP>
int launch_attn(const AttnParams& p, const AttnPlan& a, int rows, cudaStream_t st) {
    if (a.split) return a.groups == 1 ? launch_split<D, SP, 1>(p, a, rows, st) : launch_split<D, SP, 2>(p, a, rows, st);
    if (a.prompt) return launch_prompt<D, SP == 2>(p, st);
    if constexpr (SP == 2) {                 // fp32 queries (a 16-bit prompt went to launch_prompt)
        static std::atomic<bool> granted[kMaxDev];
        const int sm = kAttnWarps * (kTileGroups<D> * 3 * (D / 32) * 256 + 128 + Ring<D>::kBytes);
        if (int rc = allow_smem(k_attn_tiles<D>, granted, sm, "kv8_attention: shared memory")) return rc;
        k_attn_check<<<1, 256, 0, st>>>(p);
        if (int rc = ccuda("kv8_attention: check")) return rc;
        // the tiles come up beside the check, on which nothing of theirs depends
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3((unsigned) ((p.tiles + kAttnWarps - 1) / kAttnWarps), p.c.H, p.n_req);
        cfg.blockDim = dim3(kAttnWarps * 32);
        cfg.dynamicSmemBytes = sm;
        cfg.stream = st;
        cudaLaunchAttribute at{};
        at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &at;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, k_attn_tiles<D>, p);
    }
    return ccuda("kv8_attention");
}

}  // namespace

// This file's copy of the bound of the waits (tsb_set_wait_limit_ns writes each).
int cache_set_wait_limit(unsigned long long ns) {
    return cudaMemcpyToSymbol(g_wait_ns, &ns, sizeof ns) == cudaSuccess ? TSB_OK : TSB_ERR_CUDA;
}

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
    static std::atomic<bool> granted[kMaxDev];
    if (int rc = allow_smem(k_block_tables, granted, 3 * (kTabMaxReq + 1) * 4, "block_tables: shared memory")) return rc;
    // a thread a token, and for blocks that may be given back
    const int64_t work = std::max<int64_t>({cap_tokens, n_req, (int64_t) n_req * table_width / 16});
    const int ctas = (int) std::min<int64_t>(std::max<int64_t>((work + kTabThreads - 1) / kTabThreads, 1), std::max(2 * sm_count(), 1));
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
    AppendParams p{cache_of(cache), k, v, elem_type, k_tok, k_head, v_tok, v_head, slots, n_tok, false};
    p.wide = !((uintptr_t) k % 16 || (uintptr_t) v % 16 || (k_tok * es) % 16 || (k_head * es) % 16 || (v_tok * es) % 16 ||
               (v_head * es) % 16);
    // Few tokens are taken for decode steps, a run each: a warp a token; many for prompts: a CTA a block's worth.  What decides
    // is the length of the runs, which only the device knows.  Measured, a warp a token against a CTA a block's worth (us,
    // 8 heads of 128, bf16, blocks of 16): requests of one token, 256 of them 4 against 29, 1024 10 against 59, 4000 31 against
    // 175; one prompt of 64 tokens 10 against 4, of 1000 12 against 8, of 4000 24 against 20.  So up to 1024 tokens a wrong guess
    // costs 2 to 6 us and is made for prompts; above, it costs most in steps of thousands of requests.
    const bool few = n_tok <= 1024;
    const int64_t ctas = few ? (n_tok + 3) / 4 : (n_tok + cache->block_size - 1) / cache->block_size;
    if (ctas > 0x7fffffffll / 2 / cache->n_kv_heads) return cfail(TSB_ERR_UNSUPPORTED, "kv8_append: too many tokens");
    const unsigned grid = (unsigned) (ctas * 2 * cache->n_kv_heads);
    if (few) k_kv8_append<<<grid, 128, 0, cst(stream)>>>(p);
    else k_kv8_append_runs<<<grid, 128, 0, cst(stream)>>>(p);
    return ccuda("kv8_append");
}

int tsb_kv8_read(const tsb_kv8* cache, const int64_t* slots, int64_t n_tok, void* k, void* v, int elem_type, void* stream) {
    if (int rc = check_cache(cache, "kv8_read")) return rc;
    if (!elem_ok(elem_type)) return cfail(TSB_ERR_UNSUPPORTED, "kv8_read: element type %d (F32, F16, BF16)", elem_type);
    if (n_tok < 0) return cfail(TSB_ERR_ARG, "kv8_read: n_tok");
    if (n_tok == 0) return TSB_OK;
    if (!k || !v || !slots) return cfail(TSB_ERR_ARG, "kv8_read: null pointer");
    if ((uintptr_t) k % 16 || (uintptr_t) v % 16) return cfail(TSB_ERR_ALIGN, "kv8_read: 16-byte aligned outputs");
    const int64_t ctas = (n_tok * (cache->head_dim / 4) + 256 * kReadSteps - 1) / (256 * kReadSteps);
    if (ctas > 0x7fffffffll / 2 / cache->n_kv_heads) return cfail(TSB_ERR_UNSUPPORTED, "kv8_read: too many tokens");
    k_kv8_read<<<(unsigned) (ctas * 2 * cache->n_kv_heads), 256, 0, cst(stream)>>>(cache_of(cache), slots, n_tok, k, v, elem_type);
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
    if (d->table_stride < 0) return cfail(TSB_ERR_ARG, "kv8_attention: table_stride");
    const int es = elem_bytes(d->elem_type);
    if ((uintptr_t) q % es || (uintptr_t) out % es) return cfail(TSB_ERR_ALIGN, "kv8_attention: element alignment");
    if (a.ws && (!workspace || ws_bytes < a.ws))
        return cfail(TSB_ERR_WORKSPACE, "kv8_attention: workspace of %llu bytes needed", (unsigned long long) a.ws);
    if (a.ws && (uintptr_t) workspace % 16) return cfail(TSB_ERR_ALIGN, "kv8_attention: 16-byte aligned workspace");
    if ((int64_t) d->n_req * cache->n_kv_heads * a.tiles > 0x7ffffffell || d->n_req > 65535)
        return cfail(TSB_ERR_UNSUPPORTED, "kv8_attention: too many requests");
    AttnParams p{};
    p.c = cache_of(cache);
    p.q = q, p.o = out, p.type = d->elem_type, p.n_req = d->n_req, p.G = a.G, p.max_q = d->max_q, p.window = d->window;
    p.scale_log2 = d->scale * 1.4426950408889634f;
    p.q_tok = d->q_tok, p.q_head = d->q_head, p.o_tok = d->o_tok, p.o_head = d->o_head, p.n_tok = d->n_tok;
    p.table = table, p.table_stride = d->table_stride, p.width = d->table_width, p.lens = lens, p.cu = cu_q;
    p.tiles = a.tiles, p.n_cta = a.n_cta, p.err = device_error_word();
    p.pre = (int64_t*) workspace;
    p.part = (float*) ((uint8_t*) workspace + (((uint64_t) d->n_req + 1) * 8 + 255) / 256 * 256);
    p.wide_out = !((uintptr_t) out % 16 || (d->o_tok * es) % 16 || (d->o_head * es) % 16);
    const int rows = (int) std::min<int64_t>((int64_t) d->max_q * a.G, 1 << 20);
    // the weights in one fp16 value only where the output's rounding is coarser
    const bool two = d->elem_type != E_BF16;
    cudaStream_t st = cst(stream);
    switch (cache->head_dim) {
        case 64: return two ? launch_attn<64, 2>(p, a, rows, st) : launch_attn<64, 1>(p, a, rows, st);
        case 128: return two ? launch_attn<128, 2>(p, a, rows, st) : launch_attn<128, 1>(p, a, rows, st);
        default: return two ? launch_attn<256, 2>(p, a, rows, st) : launch_attn<256, 1>(p, a, rows, st);
    }
}

}  // extern "C"
