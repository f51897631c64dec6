// tsb_delta.cu - the gated delta rule: per value head a state S [dim_k][dim_v] (fp32) and per token
//     S <- e^g S;   u = beta (v - S^T k);   S <- S + k u^T;   o = scale S^T q.
// Three kernels: k_delta_step runs the recurrence itself (single tokens, short steps); for prompts k_delta_prepare turns
// chunks of 64 tokens into small triangular systems, all chunks at once, and k_delta_scan walks a sequence's chunks.
//
// A chunk with S at its start, gc the running sum of g inside it, K, Q [64][dim_k], V [64][dim_v]:
//     A_ij = beta_i e^(gc_i - gc_j) k_i . k_j for j < i           (the tokens' effect on one another)
//     M    = (1 + A)^-1 diag(beta)
//     U    = M (V - diag(e^gc) K S)                                (every token's u)
//     O    = scale (diag(e^gc) Q S + P U),  P_ij = e^(gc_i - gc_j) q_i . k_j for j <= i
//     S   <- e^gc_63 S + (diag(e^(gc_63 - gc)) K)^T U
// Only exponents of differences gc_i - gc_j with i >= j appear, so nothing overflows for g <= 0 however long the chunk
// decays; the running sums are carried in 64 bits because those differences are small numbers between large ones.
#include "../../include/tsb_moe.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <type_traits>

#include "tsb_device.cuh"
#include "tsb_warp_mma.cuh"

namespace tsb {

void set_last_error(const char* msg);   // tsb_moe.cu: the text tsb_last_error returns
unsigned* device_error_word();          // tsb_moe.cu: the current device's error word
int sm_count();                         // tsb_cache.cu: the current device's multiprocessors

namespace {

int dfail(int code, const char* fmt, ...) {
    char b[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(b, sizeof b, fmt, ap);
    va_end(ap);
    set_last_error(b);
    return code;
}
int dcuda(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return dfail(TSB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    return TSB_OK;
}

constexpr int kChunk = 64;
constexpr float kFinite = 3.4028235e38f;         // the largest finite value
constexpr uint32_t kFiniteBits = 0x7f7fffffu;
#define kNaN __uint_as_float(0x7fffffffu)
constexpr unsigned kSiteDelta = 0xD0000001u;   // the error word when the scan's wait for a chunk's tiles gave up,
constexpr unsigned kSiteState = 0xD0000002u;   // when state_idx names a state that there is not,
constexpr unsigned kSiteLong = 0xD0000003u;    // and when a sequence is longer than max_len or reaches past n_tok

struct DeltaParams {
    const void *q, *k, *v;
    const float *g, *beta;
    const float* s_in;
    float* s_out;
    const int32_t* idx;              // state of each sequence (null: its number); negative: from zeros, not kept
    const int32_t* cu;               // null: n_seq sequences of max_len tokens
    void* o;
    int type, n_seq, max_len, hk, hv, dk, dv, n_states;
    int64_t n_tok;
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head, gb_tok;
    float scale, eps;
    bool norm, wide;                 // q and k to unit length first; 16-byte loads allowed
    // prompts
    uint8_t* ws;
    int max_chunks;
    unsigned* err;
};

struct Seq {
    int64_t tok;
    int n;
};
__device__ __forceinline__ Seq seq_of(const DeltaParams& p, int b) {
    Seq s;
    if (p.cu) {
        s.tok = max(p.cu[b], 0);
        const int64_t end = min((int64_t) p.cu[b + 1], p.n_tok);
        s.n = (int) max((int64_t) 0, min(end - s.tok, (int64_t) p.max_len));
    } else {
        s.tok = (int64_t) b * p.max_len;
        s.n = p.max_len;
    }
    return s;
}
// The sequence's state: -1 none (negative, or not one of the caller's states).
__device__ __forceinline__ int state_of(const DeltaParams& p, int b) {
    const int i = p.idx ? p.idx[b] : b;
    return i >= 0 && i < p.n_states ? i : -1;
}
// What the device's own counts ask beyond the caller's sizes is left out, and said in the error word.
__device__ __forceinline__ void check_sequence(const DeltaParams& p, int b) {
    if (p.idx && p.idx[b] >= p.n_states) report_error(p.err, kSiteState);
    if (p.cu && (int64_t) p.cu[b + 1] > min((int64_t) max(p.cu[b], 0) + p.max_len, p.n_tok)) report_error(p.err, kSiteLong);
}

// ------------------------------------------------------------------------------------------------ recurrence
__device__ __forceinline__ float4 ld_state(const float* p) {     // volatile: issued where it stands
    float4 v;
    asm volatile("ld.global.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}
// CTA (32 value columns, value head, sequence): the state's slice in registers, thread (row group of 32, 4 columns):
// dim_k / 32 rows of four columns.  One reduction over dim_k a token: S^T k and S^T q of the decayed state together,
// o = scale (S^T q + (q . k) u), so the second product needs no second pass.  Single tokens are bound by the state's
// bytes, read and written once: 128 of them with 32 heads of 128 x 128 (540 MB) take 100 to 106 us a pass on different boards, 5.1
// to 5.4 TB/s (119 while every thread summed the warps' parts for its columns, which one warp does now); 5 and 6 CTAs a SM
// measured 105 and 111 against 103.
template <int DK>
__global__ void __launch_bounds__(256, 4) k_delta_step(const DeltaParams p) {
    constexpr int RPT = DK / 32;
    __shared__ float qk[2][DK];
    __shared__ __align__(16) float red[8][2][32];
    __shared__ float dots[8][3];
    __shared__ __align__(16) float us[32];
    __shared__ float fade;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c4 = (tid & 7) * 4, rg = tid >> 3;
    const int col = blockIdx.x * 32 + c4, h = blockIdx.y, b = blockIdx.z;
    const int st = state_of(p, b);
    const int hk = h / (p.hv / p.hk);
    const int64_t base = ((int64_t) max(st, 0) * p.hv + h) * DK * p.dv + col;
    const bool in = col < p.dv;      // dim_v is a multiple of 16, so 4 columns are inside or outside together
    float4 S[RPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
        S[i] = st >= 0 && in ? ld_state(p.s_in + base + (int64_t) (i * 32 + rg) * p.dv) : make_float4(0, 0, 0, 0);
    const Seq s = seq_of(p, b);      // after the state's loads are on their way: nothing before them waits for memory
    if (blockIdx.x == 0 && h == 0 && tid == 0) check_sequence(p, b);
    if (s.n == 0 && p.s_in == p.s_out) return;
    for (int t = 0; t < s.n; ++t) {
        const int64_t tok = s.tok + t;
        float dkk = 0.0f, dqq = 0.0f, dqk = 0.0f;
        if (tid < DK) {
            const float qv = load_elem(p.q, tok * p.q_tok + (int64_t) hk * p.q_head + tid, p.type);
            const float kv = load_elem(p.k, tok * p.k_tok + (int64_t) hk * p.k_head + tid, p.type);
            qk[0][tid] = qv, qk[1][tid] = kv;
            dkk = kv * kv, dqq = qv * qv, dqk = qv * kv;
        }
        // the last warp's lanes have a column each: its value, and below its u and its output
        const int mine = blockIdx.x * 32 + lane;
        const bool finish = warp == 7, col_in = mine < p.dv;
        float v = 0.0f, g = 0.0f, beta = 0.0f;
        if (finish) {
            if (col_in) v = load_elem(p.v, tok * p.v_tok + (int64_t) h * p.v_head + mine, p.type);
            g = p.g[tok * p.gb_tok + h], beta = p.beta[tok * p.gb_tok + h];
        }
        dkk = warp_sum(dkk), dqq = warp_sum(dqq), dqk = warp_sum(dqk);
        if (lane == 0) dots[warp][0] = dkk, dots[warp][1] = dqq, dots[warp][2] = dqk;
        __syncthreads();
        float sk[4] = {0, 0, 0, 0}, sq[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const float qv = qk[0][i * 32 + rg], kv = qk[1][i * 32 + rg];
            sk[0] = fmaf(S[i].x, kv, sk[0]), sk[1] = fmaf(S[i].y, kv, sk[1]);
            sk[2] = fmaf(S[i].z, kv, sk[2]), sk[3] = fmaf(S[i].w, kv, sk[3]);
            sq[0] = fmaf(S[i].x, qv, sq[0]), sq[1] = fmaf(S[i].y, qv, sq[1]);
            sq[2] = fmaf(S[i].z, qv, sq[2]), sq[3] = fmaf(S[i].w, qv, sq[3]);
        }
        // over the row groups of a warp: a lane keeps half of what it has at each of the two steps
        const bool hi = lane & 8, odd = lane & 16;
        float k4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) k4[j] = (hi ? sq[j] : sk[j]) + __shfl_xor_sync(0xffffffffu, hi ? sk[j] : sq[j], 8);
        float k2[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) k2[j] = (odd ? k4[2 + j] : k4[j]) + __shfl_xor_sync(0xffffffffu, odd ? k4[j] : k4[2 + j], 16);
        *(float2*) &red[warp][hi][c4 + (odd ? 2 : 0)] = make_float2(k2[0], k2[1]);
        __syncthreads();
        if (finish) {
            float kk = 0.0f, qq = 0.0f, qdk = 0.0f, a = 0.0f, c = 0.0f;
#pragma unroll
            for (int w = 0; w < DK / 32; ++w) kk += dots[w][0], qq += dots[w][1], qdk += dots[w][2];
#pragma unroll
            for (int w = 0; w < 8; ++w) a += red[w][0][lane], c += red[w][1][lane];
            const float rk = p.norm ? rsqrtf(kk + p.eps) : 1.0f, rq = p.norm ? rsqrtf(qq + p.eps) : 1.0f, decay = expf(g);
            const float u = beta * (v - decay * rk * a);
            us[lane] = u * rk;
            if (lane == 0) fade = decay;
            if (col_in) store_elem(p.o, tok * p.o_tok + (int64_t) h * p.o_head + mine, p.type, p.scale * rq * (decay * c + qdk * rk * u));
        }
        __syncthreads();
        const float4 u = *(const float4*) (us + c4);
        const float decay = fade;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const float kv = qk[1][i * 32 + rg];
            S[i].x = fmaf(kv, u.x, S[i].x * decay), S[i].y = fmaf(kv, u.y, S[i].y * decay);
            S[i].z = fmaf(kv, u.z, S[i].z * decay), S[i].w = fmaf(kv, u.w, S[i].w * decay);
        }
        if (t + 1 < s.n) __syncthreads();
    }
    if (st >= 0 && in) {
#pragma unroll
        for (int i = 0; i < RPT; ++i) __stcs((float4*) (p.s_out + base + (int64_t) (i * 32 + rg) * p.dv), S[i]);
    }
}

// ------------------------------------------------------------------------------------------------ chunks
// Matrix products on 16-bit operands at fp32 accuracy: a row of an operand (the values that one result sums over) is
// scaled by a power of two that brings its largest magnitude to [2^14, 2^15) and stored as fp16, or as two fp16 values
// (x = hi + lo, 22 bits; products hi hi + lo hi + hi lo).  The result is scaled back in fp32.  bf16 and fp16 inputs are
// exact in one value down to 2^-32 of their row's largest; fp32 inputs and everything computed here take two.
// (bf16 pairs hold 16 bits: the same products left the states 8e-6 off, 2e-7 with these.)
//
// What k_delta_prepare leaves for k_delta_scan, tiles of fp16 [64 rows][row bytes] whose 16-byte pieces are permuted within
// a row (piece ^ row % 8), so that ldmatrix reads them without bank conflicts straight after a bulk copy:
//   per (chunk, key head):   K planes, Q planes [PL][64][DK]
//   per (chunk, value head): M hi, M lo [64][64], P planes [PP][64][64], then fp32 vectors [6][64]:
//     e^gc by K's row scale | scale e^gc by Q's | e^(gc_63 - gc) by K's | M's row scale | P's | e^gc_63
template <int E, int DK>
struct Tiles {
    static constexpr int PL = E == E_F32 ? 2 : 1;            // planes of K and Q
    static constexpr int PP = E == E_BF16 ? 1 : 2;           // planes of what only the output sees: 11 bits for bf16
    static constexpr int kTile = kChunk * DK * 2;
    static constexpr int kHead = 2 * PL * kTile;             // per key head
    static constexpr int kSq = kChunk * kChunk * 2;
    static constexpr int kVal = (2 + PP) * kSq + 6 * kChunk * 4;
    static constexpr int kStage = kHead + kVal;
    __host__ __device__ static int64_t chunk_bytes(int hk, int hv) { return (int64_t) hk * kHead + (int64_t) hv * kVal; }
};
enum { V_EK = 0, V_EQ = 64, V_ED = 128, V_FM = 192, V_FP = 256, V_END = 320 };

__device__ __forceinline__ uint32_t swz(int row, int piece, int row_bytes) {
    return (uint32_t) (row * row_bytes + ((piece ^ (row & 7)) << 4));
}
// The power of two that brings `peak` to [2^14, 2^15), and its inverse (peak 0 or below 2^-112: the largest of them).
__device__ __forceinline__ void pow2_scale(float peak, float& up, float& inv) {
    const int e = max((int) (__float_as_uint(peak) >> 23) & 255, 15);
    up = __uint_as_float((uint32_t) (268 - e) << 23);
    inv = __uint_as_float((uint32_t) (e - 14) << 23);
}
__device__ __forceinline__ float pow2f(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float max4(float a, float b, float c, float d) {
    return fmaxf(fmaxf(fabsf(a), fabsf(b)), fmaxf(fabsf(c), fabsf(d)));
}
// The largest of a, |x| and |y|, NaN if any is.
__device__ __forceinline__ float max_nan(float a, float x, float y) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(x)), "f"(fabsf(y)));
    return r;
}
__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ void split_f16(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    hi = pack_f16(x0, x1);
    const float2 h = __half22float2(*(const __half2*) &hi);
    lo = pack_f16(x0 - h.x, x1 - h.y);
}
// The same of u x0, u x1 (packed fp32 arithmetic).
__device__ __forceinline__ void split_f16x2(float x0, float x1, float u, uint32_t& hi, uint32_t& lo) {
    const float2 y = __fmul2_rn(make_float2(x0, x1), make_float2(u, u));
    hi = pack_f16(y.x, y.y);
    const float2 h = __half22float2(*(const __half2*) &hi);
    const float2 d = __ffma2_rn(h, make_float2(-1.0f, -1.0f), y);
    lo = pack_f16(d.x, d.y);
}
template <int E>
using Elem = std::conditional_t<E == E_F32, float, std::conditional_t<E == E_F16, __half, __nv_bfloat16>>;
template <int E>
__device__ __forceinline__ void store_t(Elem<E>* p, float v) {
    if constexpr (E == E_F32) *p = v;
    else if constexpr (E == E_F16) *p = __float2half_rn(v);
    else *p = __float2bfloat16_rn(v);
}

// Chunks before sequence b (every thread of the CTA gets the sum; n_seq is at most a few thousand).
__device__ __forceinline__ int chunks_before(const DeltaParams& p, int b, int* sh) {
    if (!p.cu) return b * ((p.max_len + kChunk - 1) / kChunk);
    int sum = 0;
    for (int i = threadIdx.x; i < b; i += blockDim.x) sum += (seq_of(p, i).n + kChunk - 1) / kChunk;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < (int) blockDim.x / 32; ++w) sum += sh[w];
    return sum;
}
// Which sequence chunk c belongs to and which of its chunks it is; false past the last chunk.
__device__ __forceinline__ bool find_chunk(const DeltaParams& p, int c, int& b, int& j, int* sh) {
    if (!p.cu) {
        const int per = (p.max_len + kChunk - 1) / kChunk;
        b = c / per, j = c % per;
        return b < p.n_seq;
    }
    if (threadIdx.x == 0) sh[0] = -1;
    __syncthreads();
    if (threadIdx.x < 32) {
        int before = 0;
        for (int s0 = 0; s0 < p.n_seq; s0 += 32) {
            const int i = s0 + threadIdx.x;
            const int n = i < p.n_seq ? (seq_of(p, i).n + kChunk - 1) / kChunk : 0;
            int v = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, o);
                if ((int) threadIdx.x >= o) v += u;
            }
            const int at = before + v - n;
            if (c >= at && c < at + n) sh[0] = i, sh[1] = c - at;
            before += __shfl_sync(0xffffffffu, v, 31);
            if (c < before) break;
        }
    }
    __syncthreads();
    b = sh[0], j = sh[1];
    return b >= 0;
}

constexpr int LA = 68;   // row pitch (floats) of the triangle and its inverse in shared memory

// In place: A21 <- -X22 (A21 X11) for the pairs of S x S blocks along the diagonal whose blocks X11, X22 are inverses
// already; 128 threads, two small fp32 products.
template <int S>
__device__ __forceinline__ void merge_blocks(float* X, float* tmp, int tid) {
    constexpr int RT = S == 32 ? 2 : 1, CT = S == 8 ? 2 : 4;       // a thread's rows and columns of the result
    constexpr int CG = S / CT, LT = S + 4;
    const int per = S * S / (RT * CT), pair = tid / per, in = tid % per;
    const int r = in / CG * RT, c = in % CG * CT, base = 2 * S * pair;
    float* T = tmp + pair * S * LT;
#pragma unroll
    for (int step = 0; step < 2; ++step) {
        const float* L = X + (base + S) * LA + base + (step == 0 ? 0 : S);
        const float* B = step == 0 ? X + base * LA + base : T;
        const int ldb = step == 0 ? LA : LT;
        float acc[RT][CT];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < CT; ++j) acc[i][j] = 0.0f;
#pragma unroll
        for (int k = 0; k < S; k += 4) {
            float4 l[RT];
#pragma unroll
            for (int i = 0; i < RT; ++i) l[i] = *(const float4*) (L + (r + i) * LA + k);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                float b[CT];
                if constexpr (CT == 4) {
                    const float4 v = *(const float4*) (B + (k + m) * ldb + c);
                    b[0] = v.x, b[1] = v.y, b[2] = v.z, b[3] = v.w;
                } else {
                    const float2 v = *(const float2*) (B + (k + m) * ldb + c);
                    b[0] = v.x, b[1] = v.y;
                }
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    const float a = m == 0 ? l[i].x : m == 1 ? l[i].y : m == 2 ? l[i].z : l[i].w;
#pragma unroll
                    for (int j = 0; j < CT; ++j) acc[i][j] = fmaf(a, b[j], acc[i][j]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < CT; ++j) {
                if (step == 0) T[(r + i) * LT + c + j] = acc[i][j];
                else X[(base + S + r + i) * LA + base + c + j] = -acc[i][j];
            }
        __syncthreads();
    }
}

// CTA (chunk, key head), four warps.  The chunk's keys and queries to fp16 planes in shared memory and in the
// workspace; K K^T and Q K^T on the tensor cores (warp w: rows 16 w); then for each value head of the key head the
// decays, A, P and M.  (1 + A)^-1 in fp32 from its 8 x 8 diagonal blocks (forward substitution, a thread a column) by
// three joins of neighbouring blocks: exact arithmetic on the triangle, where powers of A would cancel, with every
// thread at work (one thread a column over all 64 rows is 2000 dependent steps: 240 us for 8192 tokens, 32 heads; now 149).
// Bound by latency: a value head's dozen steps lie between barriers, issue slots are 29% active, and a warp waits 3.7 cycles an
// instruction for shared and 3.6 for global memory (16-bit forms spill some 140 bytes at 128 registers).
template <int E, int DK>
__global__ void __launch_bounds__(128, E == E_F32 ? 2 : 4) k_delta_prepare(const DeltaParams p) {
    using T = Tiles<E, DK>;
    constexpr int PL = T::PL, PP = T::PP;
    extern __shared__ __align__(1024) uint8_t sm[];
    uint8_t* kt = sm;                                    // [PL][64][DK]; later M and P planes and the vectors
    uint8_t* qt = sm + PL * T::kTile;
    constexpr int kStageOut = T::kVal > T::kHead ? T::kVal : T::kHead;
    float* A = (float*) (sm + kStageOut);                // [64][LA]: the triangle, inverted in place
    float* tmp = A + kChunk * LA;                        // [32][36]
    __shared__ __align__(16) float rk[kChunk], rq[kChunk], beta[kChunk];
    __shared__ __align__(16) double gc[kChunk];
    __shared__ bool k_lost[kChunk];
    __shared__ uint32_t lost[4];
    __shared__ int sh[8];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hk = blockIdx.y, rep = p.hv / p.hk;
    int b, j;
    if (!find_chunk(p, blockIdx.x, b, j, sh)) return;
    const Seq s = seq_of(p, b);
    const int live = min(kChunk, s.n - j * kChunk);
    const int64_t tok0 = s.tok + (int64_t) j * kChunk;
    uint8_t* out = p.ws + (int64_t) blockIdx.x * T::chunk_bytes(p.hk, p.hv);

    // a thread holds 8 values of a row; DK / 8 neighbouring threads a row
    constexpr int TPR = DK / 8;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const void* src = w ? p.q : p.k;
        const int64_t st = w ? p.q_tok : p.k_tok, hd = (w ? p.q_head : p.k_head) * hk;
        uint8_t* dst = w ? qt : kt;
        constexpr int NB = E == E_F32 ? 2 : 4;            // rows a thread has in flight
        for (int e0 = tid; e0 < kChunk * TPR; e0 += 128 * NB) {
            float x[NB][8];
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int e = e0 + 128 * i, row = e / TPR, piece = e % TPR;
                if (row < live) {
                    load8(x[i], src, (tok0 + row) * st + hd + piece * 8, E, p.wide);
                } else {
#pragma unroll
                    for (int m = 0; m < 8; ++m) x[i][m] = 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int e = e0 + 128 * i, row = e / TPR, piece = e % TPR;
                float sq = 0.0f, len = 1.0f;
                uint32_t peak = 0;                        // by bits: above every finite value for NaN as for infinity
#pragma unroll
                for (int m = 0; m < 8; ++m) peak = max(peak, __float_as_uint(x[i][m]) & 0x7fffffffu);
#pragma unroll
                for (int o = TPR / 2; o > 0; o >>= 1) peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, o));
                if (p.norm) {
#pragma unroll
                    for (int m = 0; m < 8; ++m) sq = fmaf(x[i][m], x[i][m], sq);
#pragma unroll
                    for (int o = TPR / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
                    if (row < live) len = rsqrtf(sq + p.eps);         // (the zeros past the last token have no length)
                }
                if (w == 0) {                             // a key that is not finite: zeros, and the head's states are lost below
                    const bool gone = peak > kFiniteBits || !(len <= kFinite);
                    if (gone) {
                        peak = 0, len = 1.0f;
#pragma unroll
                        for (int m = 0; m < 8; ++m) x[i][m] = 0.0f;
                    }
                    if (piece == 0) k_lost[row] = gone;
                }
                float up, inv;
                pow2_scale(__uint_as_float(peak), up, inv);
                if (piece == 0) (w ? rq : rk)[row] = len * inv;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int m = 0; m < 4; ++m) split_f16(x[i][2 * m] * up, x[i][2 * m + 1] * up, hi[m], lo[m]);
                const uint32_t at = swz(row, piece, DK * 2);
                *(uint4*) (dst + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if (PL == 2) *(uint4*) (dst + T::kTile + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    }
    __syncthreads();
    {
        uint4* o = (uint4*) (out + (int64_t) hk * T::kHead);
        for (int e = tid; e < T::kHead / 16; e += 128) o[e] = ((const uint4*) sm)[e];
    }
    float kk[8][4], qk[8][4];
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) kk[n][e] = qk[n][e] = 0.0f;
    const uint32_t ks = smem_u32(kt), qs = smem_u32(qt);
    const int ar = warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;       // left operand: rows of the warp
    const int br = (lane & 7) + (lane >> 4) * 8;                          // right operand: 16 tokens a load
#pragma unroll
    for (int d = 0; d < DK / 16; ++d) {
        uint32_t ak[PL][4], aq[PL][4];
#pragma unroll
        for (int l = 0; l < PL; ++l) {
            ldsm4(ak[l], ks + l * T::kTile + swz(ar, 2 * d + (lane >> 4), DK * 2));
            ldsm4(aq[l], qs + l * T::kTile + swz(ar, 2 * d + (lane >> 4), DK * 2));
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            if (n > warp) continue;                                       // above the diagonal
#pragma unroll
            for (int l = 0; l < PL; ++l) {
                uint32_t r[4];
                ldsm4(r, ks + l * T::kTile + swz(n * 16 + br, 2 * d + ((lane >> 3) & 1), DK * 2));
#pragma unroll
                for (int a = 0; a < PL - l; ++a) {                        // hi hi, lo hi, hi lo
                    mma_f16(kk[2 * n], ak[a], r[0], r[1]);
                    mma_f16(kk[2 * n + 1], ak[a], r[2], r[3]);
                    mma_f16(qk[2 * n], aq[a], r[0], r[1]);
                    mma_f16(qk[2 * n + 1], aq[a], r[2], r[3]);
                }
            }
        }
    }
    const int g = lane >> 2, qd = lane & 3;
    uint8_t* stage = sm;
    float* vec = (float*) (stage + (2 + PP) * T::kSq);
    // threads 0..63 hold a token's g, 64..127 its beta, one head ahead of their use
    const int tt = tid & 63;
    const float* gsrc = (tid < 64 ? p.g : p.beta) + (tok0 + tt) * p.gb_tok + hk * rep;
    float gnext = tt < live ? gsrc[0] : 0.0f;
    for (int i = 0; i < rep; ++i) {
        const int h = hk * rep + i;
        __syncthreads();                                  // the tiles, or the previous head's planes, are out
        // A token whose key, decay or beta is not finite (a decay of -inf is) leaves a state without a finite value, and outputs
        // from itself on.  In the products it would reach the chunk's earlier tokens too, as 0 * NaN above the diagonals; so
        // it takes part as zeros, and what it spoils is marked in the vectors.
        const bool gone = tt < live && (tid < 64 ? k_lost[tt] || !(gnext <= kFinite) : !(fabsf(gnext) <= kFinite));
        const unsigned any = __ballot_sync(0xffffffffu, gone);
        if (lane == 0) lost[warp] = any;
        // e^-200 is 0 in fp32; a sum of -inf would make differences undefined
        if (tid < 64) gc[tt] = gone ? 0.0 : (double) fmaxf(gnext, -200.0f);
        else beta[tt] = gone ? 0.0f : gnext;
        if (i + 1 < rep && tt < live) gnext = gsrc[i + 1];
        __syncthreads();
        if (warp == 0) {                                  // running sums, in units of log 2
            double v[2];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                v[w] = gc[w * 32 + lane] * 1.4426950408889634;
#pragma unroll
                for (int o2 = 1; o2 < 32; o2 <<= 1) {
                    const double u = __shfl_up_sync(0xffffffffu, v[w], o2);
                    if (lane >= o2) v[w] += u;
                }
            }
            v[1] += __shfl_sync(0xffffffffu, v[0], 31);
            const double last = __shfl_sync(0xffffffffu, v[1], 31);
            const unsigned l0 = lost[0] | lost[2], l1 = lost[1] | lost[3];
            const int from = l0 ? __ffs(l0) - 1 : l1 ? __ffs(l1) + 31 : kChunk;        // the first lost token
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const int t = w * 32 + lane;
                gc[t] = v[w];
                const float e = pow2f((float) v[w]);
                vec[V_EK + t] = e * rk[t];
                vec[V_EQ + t] = t < from ? e * rq[t] * p.scale : kNaN;
                vec[V_ED + t] = pow2f((float) (last - v[w])) * rk[t];
                vec[V_END + t] = from == kChunk ? pow2f((float) last) : kNaN;
            }
        }
        __syncthreads();
        float pv[8][4], peak[2] = {0.0f, 0.0f};
        const int row0 = warp * 16 + g;
        const double gr[2] = {gc[row0], gc[row0 + 8]};
        const float ar2[2] = {beta[row0] * rk[row0], beta[row0 + 8] * rk[row0 + 8]};
        const float pr[2] = {rq[row0] * p.scale, rq[row0 + 8] * p.scale};
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int c = n * 8 + 2 * qd;
            if (n > 2 * warp + 1) {                       // above the diagonal: the joins read zeros there, P is not read
                *(float2*) (A + row0 * LA + c) = *(float2*) (A + (row0 + 8) * LA + c) = make_float2(0.0f, 0.0f);
                continue;
            }
            const double2 gcc = *(const double2*) (gc + c);
            const float2 rc = *(const float2*) (rk + c);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = row0 + e * 8;
                const float f0 = c <= row ? pow2f((float) (gr[e] - gcc.x)) * rc.x : 0.0f;
                const float f1 = c + 1 <= row ? pow2f((float) (gr[e] - gcc.y)) * rc.y : 0.0f;
                *(float2*) (A + row * LA + c) = make_float2(c < row ? ar2[e] * (f0 * kk[n][2 * e]) : 0.0f,
                                                            c + 1 < row ? ar2[e] * (f1 * kk[n][2 * e + 1]) : 0.0f);
                pv[n][2 * e] = f0 * (pr[e] * qk[n][2 * e]);
                pv[n][2 * e + 1] = f1 * (pr[e] * qk[n][2 * e + 1]);
                peak[e] = fmaxf(peak[e], fmaxf(fabsf(pv[n][2 * e]), fabsf(pv[n][2 * e + 1])));
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = row0 + e * 8;
            float up, inv;
            pow2_scale(quad_max(peak[e]), up, inv);
            if (qd == 0) vec[V_FP + row] = inv;
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                if (n > 2 * warp + 1) continue;
                uint32_t hi, lo;
                split_f16(pv[n][2 * e] * up, pv[n][2 * e + 1] * up, hi, lo);
                const uint32_t at = swz(row, n, kChunk * 2) + qd * 4;
                *(uint32_t*) (stage + 2 * T::kSq + at) = hi;
                if (PP == 2) *(uint32_t*) (stage + 3 * T::kSq + at) = lo;
            }
        }
        __syncthreads();
        if (tid < kChunk) {                               // 8 x 8 diagonal blocks; a block's threads are in one warp
            const int o = tid & ~7, c = tid & 7;
            float x[8], w[8][8];
#pragma unroll
            for (int r = 1; r < 8; ++r)
#pragma unroll
                for (int m = 0; m < r; ++m) w[r][m] = A[(o + r) * LA + o + m];
            __syncwarp();
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                float a = r == c ? 1.0f : 0.0f;
#pragma unroll
                for (int m = 0; m < r; ++m) a = fmaf(-w[r][m], x[m], a);
                x[r] = a;
                A[(o + r) * LA + o + c] = a;
            }
        }
        __syncthreads();
        merge_blocks<8>(A, tmp, tid);
        merge_blocks<16>(A, tmp, tid);
        merge_blocks<32>(A, tmp, tid);
        {
            const int row = tid >> 1, c0 = (tid & 1) * 8;  // pieces c0, c0 + 16, ... up to the row's diagonal tile
            float m[4][8], top = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (16 * t > row) break;
#pragma unroll
                for (int c = 0; c < 8; c += 4) {
                    const float4 x = *(const float4*) (A + row * LA + 16 * t + c0 + c), w = *(const float4*) (beta + 16 * t + c0 + c);
                    m[t][c] = x.x * w.x, m[t][c + 1] = x.y * w.y, m[t][c + 2] = x.z * w.z, m[t][c + 3] = x.w * w.w;
                    top = fmaxf(top, max4(m[t][c], m[t][c + 1], m[t][c + 2], m[t][c + 3]));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            float up, inv;
            pow2_scale(top, up, inv);
            if (c0 == 0) vec[V_FM + row] = inv;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                if (16 * t > row) break;
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) split_f16(m[t][2 * u] * up, m[t][2 * u + 1] * up, hi[u], lo[u]);
                const uint32_t at = swz(row, (16 * t + c0) >> 3, kChunk * 2);
                *(uint4*) (stage + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *(uint4*) (stage + T::kSq + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        __syncthreads();
        uint4* o = (uint4*) (out + (int64_t) p.hk * T::kHead + (int64_t) h * T::kVal);
        for (int e = tid; e < T::kVal / 16; e += 128) o[e] = ((const uint4*) stage)[e];
    }
}

// Barriers of the warps that share 16 value columns (two units a CTA): the two that carry the state; those and the two that
// write the outputs; and the latter's word to the former that they have read the state.
__device__ __forceinline__ void pair_sync(int unit) { asm volatile("bar.sync %0, 64;" ::"r"(1 + unit) : "memory"); }
__device__ __forceinline__ void unit_sync(int unit) { asm volatile("bar.sync %0, 128;" ::"r"(3 + unit) : "memory"); }
// The same barriers, and whether any of their threads says so.
template <int N>
__device__ __forceinline__ bool sync_any(int id, bool x) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 q, %2, 0;\n bar.red.or.pred p, %1, %3, q;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(r) : "r"(id), "r"((uint32_t) x), "n"(N) : "memory");
    return r != 0;
}
__device__ __forceinline__ bool pair_any(int unit, bool x) { return sync_any<64>(1 + unit, x); }
__device__ __forceinline__ bool unit_any(int unit, bool x) { return sync_any<128>(3 + unit, x); }
__device__ __forceinline__ void read_sync(int unit) { asm volatile("bar.sync %0, 128;" ::"r"(5 + unit) : "memory"); }
__device__ __forceinline__ void read_arrive(int unit) { asm volatile("bar.arrive %0, 128;" ::"r"(5 + unit) : "memory"); }

// The power-of-two scales of a left operand's rows g and g + 8, and their inverses: largest magnitudes in [2^9, 2^10), so
// that the next chunk's may grow 32-fold.
struct RowScale {
    float u[2] = {0.0f, 0.0f}, i[2] = {0.0f, 0.0f};
    __device__ __forceinline__ void set(float a, float c) {
        pow2_scale(a, u[0], i[0]);
        pow2_scale(c, u[1], i[1]);
        u[0] *= 0.03125f, u[1] *= 0.03125f, i[0] *= 32.0f, i[1] *= 32.0f;
    }
    // Whether rows (or one lane's part of them) with these largest magnitudes fit fp16 pairs under the scales at full accuracy: at most 2^15, and not
    // so small that the low halves (multiples of 2^-24) lose bits.
    __device__ __forceinline__ bool holds(float a, float c) const {
        const float x = a * u[0], y = c * u[1];
        return x <= 32768.0f && y <= 32768.0f && (x >= 0.25f || a == 0.0f) && (y >= 0.25f || c == 0.0f);
    }
};

// CTA (value columns, value head, sequence).  A unit is 16 value columns, held by W warps: S^T [16][DK] stays in their
// registers in accumulator layout, which is the left operand's layout, and a chunk is five chained products
//   Y^T = S^T K^T, Z^T = S^T Q^T, U^T = (V^T - e^gc Y^T) M^T, O^T = e^gc Z^T + U^T P^T, S^T = e^gc_63 S^T + U'^T K
// whose right operands are the chunk's tiles (bulk copies, two chunks deep).  W 1: a warp owns its unit and exchanges
// nothing, eight units a CTA; W 2: the warps take half of every product's columns (tokens, keys) each and pass the left
// operands through shared memory, two units a CTA; operands are written under the scales of the chunk before, and again
// in the rare case that a row outgrew them, so that an exchange is one barrier.  Two more warps a unit (the writers) take
// Z and O, which no later chunk waits for, from the same exchanges, and bring V.  What bounds it: a sequence's chunks
// follow one another, and a unit's 400 products of 16 x 8 x 16 a chunk (bf16, dim_k 128) at 8 cycles each.  One sequence
// of 32 heads has 256 units, so W 2 puts them on 128 SMs with every scheduler at work; with more sequences W 1 does the
// same work without exchanges.  8192 tokens of 32 heads, bf16: 314 us, a chunk in some 4460 cycles.  (Stamped when it took 329:
// 4670 cycles, of which the products before the next chunk took 2140 and the exchanges 1590.)
// W 2 at dim_k 128 fills a SM's shared memory with one CTA, and is told so: with the 128 registers that two would leave it
// 8192 tokens take 504 us a pass, with 231 466.  The other forms are left to the compiler (W 1 told the same: 304 against
// 286 for 4 sequences of 1000 in fp32).
template <int DK, int W>
constexpr int kScanCtas = W == 2 && DK == 128 ? 1 : 0;
template <int E, int DK, int W>
__global__ void __launch_bounds__(256, kScanCtas<DK, W>) k_delta_scan(const DeltaParams p) {
    using T = Tiles<E, DK>;
    constexpr int PL = T::PL;
    constexpr bool OS = T::PP == 2;
    constexpr int UN = W == 1 ? 8 : 2;                 // units of a CTA
    constexpr int NK = DK / 8 / W, NP = 4 / W;         // a warp's key tiles of 8, token tiles of 16
    constexpr int NS = NK / 2 < 2 ? NK / 2 : 2;
    constexpr int kFrag = W == 1 ? 0 : 12 * 1024;      // a unit's exchanged left operands
    constexpr int RB = DK * 2, SB = kChunk * 2;        // row bytes of the key and of the square tiles
    extern __shared__ __align__(1024) uint8_t sm[];
    __shared__ uint64_t full[2], empty[2];
    __shared__ int sh[8];
    __shared__ float peaks[UN][4][W][16];
    __shared__ int lost[UN][16];                       // a column's first token (of the sequence) whose X is not finite
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, qd = lane & 3;
    const bool writer = W == 2 && warp >= 4;           // W 2: warps 0-3 carry the states of two units, 4-7 write the outputs
    const int unit = (warp & (UN * W - 1)) / W, part = warp % W;
    const int h = blockIdx.y, b = blockIdx.z, hk = h / (p.hv / p.hk);
    const Seq s = seq_of(p, b);
    const int st = state_of(p, b);
    const int first = chunks_before(p, b, sh);
    // bounds that overlap name more chunks than there are tiles for: those are left out
    const int chunks = min((s.n + kChunk - 1) / kChunk, max(p.max_chunks - first, 0));
    const int n0 = (blockIdx.x * UN + unit) * 16;
    const bool in = n0 < p.dv;                  // dim_v is a multiple of 16
    uint4* fs = (uint4*) (sm + 2 * T::kStage + unit * kFrag);   // S [DK / 16][2][32]; later U e^(gc_63 - gc) [4][2][32]
    uint4* fu = fs + 256;                                       // U [4][2][32]
    uint4* fx = fs + 512;                                       // X [4][2][32]
    if (tid < UN * 16) (&lost[0][0])[tid] = INT_MAX;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 8);
        fence_mbar_init();
        if (blockIdx.x == 0 && h == 0) check_sequence(p, b);
    }
    __syncthreads();
    const int64_t cb = T::chunk_bytes(p.hk, p.hv);
    auto fetch = [&](int c) {
        const int i = c & 1;
        const uint8_t* src = p.ws + (int64_t) (first + c) * cb;
        mbar_expect_tx(&full[i], T::kStage);
        bulk_g2s(sm + i * T::kStage, src + (int64_t) hk * T::kHead, T::kHead, &full[i]);
        bulk_g2s(sm + i * T::kStage + T::kHead, src + (int64_t) p.hk * T::kHead + (int64_t) h * T::kVal, T::kVal, &full[i]);
    };
    const bool fetches = tid == (W == 1 ? 0 : 128);
    if (fetches) {
        for (int c = 0; c < min(chunks, 2); ++c) fetch(c);
    }
    // a warp's token tiles: with two warps 0, 3 and 1, 2, which share the triangles' work evenly
    auto tile_of = [&](int x) { return W == 1 ? x : x == 0 ? part : 3 - part; };
    float S[NK][4];
    const int64_t base = ((int64_t) max(st, 0) * p.hv + h) * DK * p.dv + n0 + (int64_t) part * NK * 8 * p.dv;
#pragma unroll
    for (int i = 0; i < NK; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            S[i][e] = st >= 0 && in && !writer ? p.s_in[base + (int64_t) (i * 8 + 2 * qd + (e & 1)) * p.dv + g + (e >> 1) * 8] : 0.0f;

    auto split_a = [&](const float (&x)[4], const float (&y)[4], const RowScale& r, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
        split_f16x2(x[0], x[1], r.u[0], hi[0], lo[0]);
        split_f16x2(x[2], x[3], r.u[1], hi[1], lo[1]);
        split_f16x2(y[0], y[1], r.u[0], hi[2], lo[2]);
        split_f16x2(y[2], y[3], r.u[1], hi[3], lo[3]);
    };
    // a row's part of a left operand (depth d of 16) into the unit's exchange, and out of it
    auto put = [&](uint4* f, int d, const float (&x)[4], const float (&y)[4], const RowScale& r) {
        uint32_t hi[4], lo[4];
        split_a(x, y, r, hi, lo);
        f[(d * 2) * 32 + lane] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        f[(d * 2 + 1) * 32 + lane] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    };
    auto get = [&](const uint4* f, int d, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
        const uint4 a = f[(d * 2) * 32 + lane], c = f[(d * 2 + 1) * 32 + lane];
        hi[0] = a.x, hi[1] = a.y, hi[2] = a.z, hi[3] = a.w;
        lo[0] = c.x, lo[1] = c.y, lo[2] = c.z, lo[3] = c.w;
    };
    // largest magnitudes of the rows g and g + 8 in the warp's part, for the unit's other warps
    auto tell_peak = [&](float& a, float& c, int kind) {
        a = quad_max(a), c = quad_max(c);
        if (W > 1 && qd == 0) peaks[unit][kind][part][g] = a, peaks[unit][kind][part][g + 8] = c;
    };
    auto join_peak = [&](float& a, float& c, int kind) {
        if constexpr (W > 1) {
#pragma unroll
            for (int w = 0; w < W; ++w) a = fmaxf(a, peaks[unit][kind][w][g]), c = fmaxf(c, peaks[unit][kind][w][g + 8]);
        }
    };
    RowScale rs, rx, ru, rf;                     // of S, X, U and U e^(gc_63 - gc)
    auto state_peak = [&](float& a, float& c) {
        a = c = 0.0f;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            a = fmaxf(a, fmaxf(fabsf(S[i][0]), fabsf(S[i][1])));
            c = fmaxf(c, fmaxf(fabsf(S[i][2]), fabsf(S[i][3])));
        }
    };
    auto put_state = [&]() {
#pragma unroll
        for (int d = 0; d < NK / 2; ++d) put(fs, part * (NK / 2) + d, S[2 * d], S[2 * d + 1], rs);
    };
    auto share_state = [&]() {
        float a, c;
        state_peak(a, c);
        if constexpr (W == 1) {
            tell_peak(a, c, 0);
            rs.set(a, c);
        } else {
            put_state();
            if (unit_any(unit, !rs.holds(a, c))) {
                tell_peak(a, c, 0);
                unit_sync(unit);
                join_peak(a, c, 0);
                rs.set(a, c);
                put_state();
                unit_sync(unit);
            }
        }
    };
    // the values of the unit's columns, as the inputs hold them until they are used
    using Raw = std::conditional_t<E == E_F32, float, uint16_t>;
    Raw V[NP * 2][4];
    const Raw* vp = (const Raw*) p.v + (int64_t) h * p.v_head + n0 + g;
    using Out = Elem<E>;
    Out* op = (Out*) p.o + (int64_t) h * p.o_head + n0 + g;
    auto load_values = [&](int c) {
        const int live = in ? min(kChunk, s.n - c * kChunk) : 0;
        const Raw* r0 = vp + (s.tok + (int64_t) c * kChunk + 2 * qd) * p.v_tok;
#pragma unroll
        for (int x = 0; x < NP; ++x) {
            const Raw* r = r0 + tile_of(x) * 16 * p.v_tok;
            const Raw* rows[2][2] = {{r, r + p.v_tok}, {r + 8 * p.v_tok, r + 9 * p.v_tok}};
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    V[2 * x + y][e] = tile_of(x) * 16 + 2 * qd + 8 * y + (e & 1) < live ? rows[y][e & 1][(e >> 1) * 8] : Raw(0);
        }
    };
    auto value = [&](Raw r) -> float {
        if constexpr (E == E_F32) return r;
        else if constexpr (E == E_F16) return __half2float(__ushort_as_half(r));
        else return __uint_as_float((uint32_t) r << 16);
    };
    // byte offsets of a lane's ldmatrix rows: right operands by rows (16 tokens a load) and transposed (keys); the
    // piece of depth d or key tile n is an xor with 32 d or 32 n
    const int br = (lane & 7) + (lane >> 4) * 8, tr = (lane & 7) + ((lane >> 3) & 1) * 8;
    const uint32_t row_x = (((lane >> 3) & 1) ^ (br & 7)) << 4, col_x = ((lane >> 4) ^ (tr & 7)) << 4;
    bool ok = true;
    // after a wait that gave up: the copies of chunks c .. to - 1 land before the CTA's memory goes
    auto land = [&](int c, int to) {
        for (; c < min(to, chunks); ++c) mbar_drain(&full[c & 1], (c >> 1) & 1, p.err, kSiteDelta);
    };
    auto wait_tiles = [&](int c) {
        if (!ok) return;
        ok = mbar_wait_bounded(&full[c & 1], (c >> 1) & 1, p.err, kSiteDelta);
        if (!ok && fetches) land(c, c + 2);
    };
    // a chunk's tiles are read by all 8 warps; then those of the chunk after the next take their place
    auto release = [&](int c) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[c & 1]);
        if (fetches && c + 2 < chunks && ok) {
            ok = mbar_wait_bounded(&empty[c & 1], (c >> 1) & 1, p.err, kSiteDelta);
            if (ok) fetch(c + 2);
            else land(c + 1, c + 2);
        }
    };
    // Z^T: tokens' states' part of the outputs
    auto scale_z = [&](float (&Z)[NP * 2][4], const float* vec) {
#pragma unroll
        for (int n = 0; n < NP * 2; ++n) {
            const float2 eq = *(const float2*) (vec + V_EQ + tile_of(n >> 1) * 16 + (n & 1) * 8 + 2 * qd);
            Z[n][0] *= eq.x * rs.i[0], Z[n][1] *= eq.y * rs.i[0], Z[n][2] *= eq.x * rs.i[1], Z[n][3] *= eq.y * rs.i[1];
        }
    };
    // X^T of chunk c with zeros for what is not finite (a value, or the state): such a token spoils its column from itself
    // on, but as 0 * NaN it would reach the tokens before it.  Also the rows' largest magnitudes.
    auto clean = [&](int c, float (&X)[NP * 2][4], float& a, float& cc) {
        a = cc = 0.0f;
#pragma unroll
        for (int n = 0; n < NP * 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!(fabsf(X[n][e]) <= kFinite)) {
                    atomicMin(&lost[unit][g + (e >> 1) * 8], c * kChunk + tile_of(n >> 1) * 16 + (n & 1) * 8 + 2 * qd + (e & 1));
                    X[n][e] = 0.0f;
                }
                if (e < 2) a = fmaxf(a, fabsf(X[n][e]));
                else cc = fmaxf(cc, fabsf(X[n][e]));
            }
    };
    // O^T = Z^T + U^T P^T of chunk c, from U's left operands
    auto outputs = [&](int c, uint32_t mr, const float* vec, float (&Z)[NP * 2][4], const uint32_t (&xh)[4][4], const uint32_t (&xl)[4][4]) {
        const int live = in ? min(kChunk, s.n - c * kChunk) : 0;
        const int from[2] = {lost[unit][g], lost[unit][g + 8]};
        if (__any_sync(0xffffffffu, min(from[0], from[1]) < (c + 1) * kChunk)) {
#pragma unroll
            for (int n = 0; n < NP * 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c * kChunk + tile_of(n >> 1) * 16 + (n & 1) * 8 + 2 * qd + (e & 1) >= from[e >> 1]) Z[n][e] = kNaN;
            __syncwarp();
        }
        float O[NP * 2][4];
#pragma unroll
        for (int n = 0; n < NP * 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) O[n][e] = 0.0f;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const uint32_t at = mr + (row_x ^ (32 * d)) + 2 * T::kSq;
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                if (d > tile_of(n)) continue;
                uint32_t r[4];
                ldsm4(r, at + tile_of(n) * 16 * SB);
                mma_f16(O[2 * n], xh[d], r[0], r[1]);
                mma_f16(O[2 * n + 1], xh[d], r[2], r[3]);
                if (OS) {
                    uint32_t w[4];
                    ldsm4(w, at + tile_of(n) * 16 * SB + T::kSq);
                    mma_f16(O[2 * n], xl[d], r[0], r[1]);
                    mma_f16(O[2 * n + 1], xl[d], r[2], r[3]);
                    mma_f16(O[2 * n], xh[d], w[0], w[1]);
                    mma_f16(O[2 * n + 1], xh[d], w[2], w[3]);
                }
            }
        }
        Out* r0 = op + (s.tok + (int64_t) c * kChunk + 2 * qd) * p.o_tok;
#pragma unroll
        for (int n = 0; n < NP * 2; ++n) {
            const int t0 = tile_of(n >> 1) * 16 + (n & 1) * 8;
            const float2 fp = *(const float2*) (vec + V_FP + t0 + 2 * qd);
            Out* r = r0 + t0 * p.o_tok;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float o = fmaf(O[n][e], (e & 1 ? fp.y : fp.x) * ru.i[e >> 1], Z[n][e]);
                Out* at = (e & 1 ? r + p.o_tok : r) + (e >> 1) * 8;
                if (t0 + 2 * qd + (e & 1) < live) store_t<E>(at, o);
            }
        }
    };
    if constexpr (W == 2) {
        if (writer) {                           // meets the same barriers as the warps that carry the states, and knows their scales
            auto meet_state = [&]() {
                if (unit_any(unit, false)) {
                    float a = 0.0f, cc = 0.0f;
                    unit_sync(unit);
                    join_peak(a, cc, 0);
                    rs.set(a, cc);
                    unit_sync(unit);
                }
            };
            // the next chunk's values to the warps that carry the states: each lane's own, where it will put its X
            auto give_values = [&]() {
#pragma unroll
                for (int n = 0; n < NP * 2; ++n)
                    ((float4*) fx)[(tile_of(n >> 1) * 2 + (n & 1)) * 32 + lane] =
                        make_float4(value(V[n][0]), value(V[n][1]), value(V[n][2]), value(V[n][3]));
            };
            if (chunks > 0) {
                load_values(0);
                give_values();
            }
            meet_state();
            for (int c = 0; c < chunks; ++c) {
                const int i = c & 1;
                if (c + 1 < chunks) load_values(c + 1);
                wait_tiles(c);
                const uint32_t kt = smem_u32(sm + i * T::kStage), mt = kt + T::kHead;
                const float* vec = (const float*) (sm + i * T::kStage + T::kHead + (2 + T::PP) * T::kSq);
                float Z[NP * 2][4];
#pragma unroll
                for (int n = 0; n < NP * 2; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) Z[n][e] = 0.0f;
#pragma unroll
                for (int d = 0; d < DK / 16; ++d) {
                    uint32_t hi[4], lo[4], rq[NP][PL][4];
#pragma unroll
                    for (int n = 0; n < NP; ++n)
#pragma unroll
                        for (int l = 0; l < PL; ++l) ldsm4(rq[n][l], kt + br * RB + (row_x ^ (32 * d)) + tile_of(n) * 16 * RB + (PL + l) * T::kTile);
                    get(fs, d, hi, lo);
#pragma unroll
                    for (int l = 0; l < PL; ++l)
#pragma unroll
                        for (int n = 0; n < NP; ++n) {
                            mma_f16(Z[2 * n], hi, rq[n][l][0], rq[n][l][1]);
                            mma_f16(Z[2 * n + 1], hi, rq[n][l][2], rq[n][l][3]);
                        }
                    if (OS) {
#pragma unroll
                        for (int n = 0; n < NP; ++n) {
                            mma_f16(Z[2 * n], lo, rq[n][0][0], rq[n][0][1]);
                            mma_f16(Z[2 * n + 1], lo, rq[n][0][2], rq[n][0][3]);
                        }
                    }
                }
                scale_z(Z, vec);
                read_arrive(unit);
                float ua = 0.0f, uc = 0.0f, fa = 0.0f, fc = 0.0f;
                unit_sync(unit);
                join_peak(ua, uc, 2);
                join_peak(fa, fc, 3);
                if (!__all_sync(0xffffffffu, ru.holds(ua, uc) && rf.holds(fa, fc))) {
                    ru.set(ua, uc);
                    rf.set(fa, fc);
                    unit_sync(unit);
                    unit_sync(unit);
                }
                if (c + 1 < chunks) give_values();
                uint32_t xh[4][4], xl[4][4];
#pragma unroll
                for (int d = 0; d < 4; ++d) get(fu, d, xh[d], xl[d]);
                outputs(c, mt + br * SB, vec, Z, xh, xl);
                release(c);
                if (c + 1 < chunks) meet_state();
            }
            return;
        }
    }
    if (W == 1 && chunks > 0) load_values(0);
    share_state();
    for (int c = 0; c < chunks; ++c) {
        const int i = c & 1;
        // after a wait that gave up the loop runs on over whatever the tiles hold, so that every barrier is met
        wait_tiles(c);
        const uint32_t kt = smem_u32(sm + i * T::kStage), mt = kt + T::kHead;
        const uint32_t kr = kt + br * RB, mr = mt + br * SB, kc = kt + tr * RB;
        const float* vec = (const float*) (sm + i * T::kStage + T::kHead + (2 + T::PP) * T::kSq);

        float Y[NP * 2][4], Z[NP * 2][4];
#pragma unroll
        for (int n = 0; n < NP * 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) Y[n][e] = Z[n][e] = 0.0f;
#pragma unroll
        for (int d = 0; d < DK / 16; ++d) {
            uint32_t hi[4], lo[4], rk[NP][PL][4], rq[NP][PL][4];
            const uint32_t at = kr + (row_x ^ (32 * d));
#pragma unroll
            for (int n = 0; n < NP; ++n)
#pragma unroll
                for (int l = 0; l < PL; ++l) {
                    ldsm4(rk[n][l], at + tile_of(n) * 16 * RB + l * T::kTile);
                    if (W == 1) ldsm4(rq[n][l], at + tile_of(n) * 16 * RB + (PL + l) * T::kTile);
                }
            if constexpr (W == 1) split_a(S[2 * d], S[2 * d + 1], rs, hi, lo);
            else get(fs, d, hi, lo);
#pragma unroll
            for (int l = 0; l < PL; ++l)
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    mma_f16(Y[2 * n], hi, rk[n][l][0], rk[n][l][1]);
                    mma_f16(Y[2 * n + 1], hi, rk[n][l][2], rk[n][l][3]);
                    if (W == 1) {
                        mma_f16(Z[2 * n], hi, rq[n][l][0], rq[n][l][1]);
                        mma_f16(Z[2 * n + 1], hi, rq[n][l][2], rq[n][l][3]);
                    }
                }
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                mma_f16(Y[2 * n], lo, rk[n][0][0], rk[n][0][1]);
                mma_f16(Y[2 * n + 1], lo, rk[n][0][2], rk[n][0][3]);
                if (W == 1 && OS) {
                    mma_f16(Z[2 * n], lo, rq[n][0][0], rq[n][0][1]);
                    mma_f16(Z[2 * n + 1], lo, rq[n][0][2], rq[n][0][3]);
                }
            }
        }
        if (W == 1) scale_z(Z, vec);
        float a = 0.0f, cc = 0.0f;
#pragma unroll
        for (int n = 0; n < NP * 2; ++n) {
            const int t = tile_of(n >> 1) * 16 + (n & 1) * 8 + 2 * qd;
            const float2 ek = *(const float2*) (vec + V_EK + t);
            float4 v;
            if constexpr (W == 1) v = make_float4(value(V[n][0]), value(V[n][1]), value(V[n][2]), value(V[n][3]));
            else v = ((const float4*) fx)[(tile_of(n >> 1) * 2 + (n & 1)) * 32 + lane];
            Y[n][0] = fmaf(-ek.x * rs.i[0], Y[n][0], v.x), Y[n][1] = fmaf(-ek.y * rs.i[0], Y[n][1], v.y);
            Y[n][2] = fmaf(-ek.x * rs.i[1], Y[n][2], v.z), Y[n][3] = fmaf(-ek.y * rs.i[1], Y[n][3], v.w);
            a = max_nan(a, Y[n][0], Y[n][1]);
            cc = max_nan(cc, Y[n][2], Y[n][3]);
        }
        bool cut = false;                           // X had to be cleaned
        if (W == 1 && c + 1 < chunks) load_values(c + 1);   // they arrive during the rest of this chunk

        uint32_t xh[4][4], xl[4][4];               // X's left operands, all token tiles; then U's
        if constexpr (W == 1) {
            cut = __any_sync(0xffffffffu, !(a <= kFinite && cc <= kFinite));
            if (cut) {
                clean(c, Y, a, cc);
                __syncwarp();
            }
            tell_peak(a, cc, 1);
            rx.set(a, cc);
#pragma unroll
            for (int d = 0; d < 4; ++d) split_a(Y[2 * d], Y[2 * d + 1], rx, xh[d], xl[d]);
        } else {
#pragma unroll
            for (int n = 0; n < NP; ++n) put(fx, tile_of(n), Y[2 * n], Y[2 * n + 1], rx);
            if (pair_any(unit, !rx.holds(a, cc))) {
                cut = true;
                clean(c, Y, a, cc);
                tell_peak(a, cc, 1);
                pair_sync(unit);
                join_peak(a, cc, 1);
                rx.set(a, cc);
#pragma unroll
                for (int n = 0; n < NP; ++n) put(fx, tile_of(n), Y[2 * n], Y[2 * n + 1], rx);
                pair_sync(unit);
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) get(fx, d, xh[d], xl[d]);
        }
        float U[NP * 2][4];
#pragma unroll
        for (int n = 0; n < NP * 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) U[n][e] = 0.0f;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t r[NP][4], w[NP][4];
            const uint32_t at = mr + (row_x ^ (32 * d));
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                if (d > tile_of(n)) continue;      // M is lower triangular
                ldsm4(r[n], at + tile_of(n) * 16 * SB);
                ldsm4(w[n], at + tile_of(n) * 16 * SB + T::kSq);
            }
#pragma unroll
            for (int x = 0; x < 3; ++x)
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    if (d > tile_of(n)) continue;
                    mma_f16(U[2 * n], x == 1 ? xl[d] : xh[d], x == 2 ? w[n][0] : r[n][0], x == 2 ? w[n][1] : r[n][1]);
                    mma_f16(U[2 * n + 1], x == 1 ? xl[d] : xh[d], x == 2 ? w[n][2] : r[n][2], x == 2 ? w[n][3] : r[n][3]);
                }
        }
        float F[NP * 2][4];                         // U e^(gc_63 - gc) by K's row scale
        float ua = 0.0f, uc = 0.0f, fa = 0.0f, fc = 0.0f;
#pragma unroll
        for (int n = 0; n < NP * 2; ++n) {
            const int t = tile_of(n >> 1) * 16 + (n & 1) * 8 + 2 * qd;
            const float2 fm = *(const float2*) (vec + V_FM + t), ed = *(const float2*) (vec + V_ED + t);
            U[n][0] *= fm.x * rx.i[0], U[n][1] *= fm.y * rx.i[0], U[n][2] *= fm.x * rx.i[1], U[n][3] *= fm.y * rx.i[1];
            F[n][0] = U[n][0] * ed.x, F[n][1] = U[n][1] * ed.y, F[n][2] = U[n][2] * ed.x, F[n][3] = U[n][3] * ed.y;
            ua = fmaxf(ua, fmaxf(fabsf(U[n][0]), fabsf(U[n][1]))), uc = fmaxf(uc, fmaxf(fabsf(U[n][2]), fabsf(U[n][3])));
            fa = fmaxf(fa, fmaxf(fabsf(F[n][0]), fabsf(F[n][1]))), fc = fmaxf(fc, fmaxf(fabsf(F[n][2]), fabsf(F[n][3])));
        }
        uint32_t fh[4][4], fl[4][4];
        tell_peak(ua, uc, 2);
        tell_peak(fa, fc, 3);
        if constexpr (W == 1) {
            ru.set(ua, uc);
            rf.set(fa, fc);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                split_a(U[2 * d], U[2 * d + 1], ru, xh[d], xl[d]);
                split_a(F[2 * d], F[2 * d + 1], rf, fh[d], fl[d]);
            }
        } else {
            auto put_u = [&]() {
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    put(fu, tile_of(n), U[2 * n], U[2 * n + 1], ru);
                    put(fs, tile_of(n), F[2 * n], F[2 * n + 1], rf);
                }
            };
            read_sync(unit);                        // the writers have read S and the last chunk's U
            put_u();
            // (by the rows' own peaks: the decay leaves most lanes of F far below theirs)
            unit_sync(unit);
            join_peak(ua, uc, 2);
            join_peak(fa, fc, 3);
            if (!__all_sync(0xffffffffu, ru.holds(ua, uc) && rf.holds(fa, fc))) {
                ru.set(ua, uc);
                rf.set(fa, fc);
                unit_sync(unit);
                put_u();
                unit_sync(unit);
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) get(fs, d, fh[d], fl[d]);
        }
        // S^T, two pairs of key tiles at a time (eight products in flight): the scaled product is added in fp32
        const float end = vec[V_END];
        const float end_f[2] = {rf.i[0], rf.i[1]};
#pragma unroll
        for (int n = 0; n < NK / 2; n += NS) {
            float acc[2 * NS][4];
#pragma unroll
            for (int x = 0; x < 2 * NS; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[x][e] = 0.0f;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                uint32_t r[NS][PL][4];
#pragma unroll
                for (int y = 0; y < NS; ++y)
#pragma unroll
                    for (int l = 0; l < PL; ++l)
                        ldsm4_t(r[y][l], kc + (col_x ^ (32 * (part * (NK / 2) + n + y))) + d * 16 * RB + l * T::kTile);
#pragma unroll
                for (int l = 0; l < PL + 1; ++l)
#pragma unroll
                    for (int y = 0; y < NS; ++y) {
                        const int k = l == 2 ? 1 : 0;            // hi hi, lo hi, hi lo
                        mma_f16(acc[2 * y], l == 1 ? fl[d] : fh[d], r[y][k * (PL - 1)][0], r[y][k * (PL - 1)][1]);
                        mma_f16(acc[2 * y + 1], l == 1 ? fl[d] : fh[d], r[y][k * (PL - 1)][2], r[y][k * (PL - 1)][3]);
                    }
            }
#pragma unroll
            for (int x = 0; x < 2 * NS; ++x)
#pragma unroll
                for (int e = 0; e < 4; ++e) S[2 * n + x][e] = fmaf(acc[x][e], end_f[e >> 1], S[2 * n + x][e] * end);
        }
        if (cut) {                                  // columns that were lost up to here have no state
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (lost[unit][g + 8 * x] >= (c + 1) * kChunk) continue;
#pragma unroll
                for (int n = 0; n < NK; ++n) S[n][2 * x] = S[n][2 * x + 1] = kNaN;
            }
        }
        if (W == 1) outputs(c, mr, vec, Z, xh, xl);
        release(c);
        if (c + 1 < chunks) {
            if (W == 2) pair_sync(unit);            // F is read
            share_state();
        }
    }
    if (ok && st >= 0 && in) {
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                p.s_out[base + (int64_t) (i * 8 + 2 * qd + (e & 1)) * p.dv + g + (e >> 1) * 8] = S[i][e];
    }
}

// ------------------------------------------------------------------------------------------------ host
// Sequences of up to this many tokens run the recurrence.  Measured, the recurrence against chunks (us, 32 heads of 128, bf16): one
// sequence of 16 tokens 17 against 27, of 24 25 against 27, of 32 32 against 28; 16 of 8 tokens 47 against 71, of 16 86 against 77;
// 64 of 8 177 against 230, of 16 331 against 248.  (The chunks' error is larger: states 3e-7 against 1e-7 of 64 bits.)
constexpr int kStepTokens = 16;

int delta_check(const tsb_delta_desc* d) {
    if (!d || d->struct_size != sizeof(tsb_delta_desc)) return dfail(TSB_ERR_ARG, "gated_delta: struct_size");
    if (d->elem_type != E_F32 && d->elem_type != E_F16 && d->elem_type != E_BF16)
        return dfail(TSB_ERR_UNSUPPORTED, "gated_delta: element type %d (F32, F16, BF16)", d->elem_type);
    if (d->n_seq < 0 || d->max_len < 0 || d->n_tok < 0 || d->n_states < 0)
        return dfail(TSB_ERR_ARG, "gated_delta: negative sizes");
    if (d->k_heads < 1 || d->v_heads < 1 || d->v_heads % d->k_heads)
        return dfail(TSB_ERR_ARG, "gated_delta: v_heads %d not a multiple of k_heads %d", d->v_heads, d->k_heads);
    if (d->dim_k != 64 && d->dim_k != 128) return dfail(TSB_ERR_UNSUPPORTED, "gated_delta: dim_k %d (64 or 128)", d->dim_k);
    if (d->dim_v < 16 || d->dim_v % 16) return dfail(TSB_ERR_UNSUPPORTED, "gated_delta: dim_v %d (a multiple of 16)", d->dim_v);
    if (d->v_heads > 65535 || d->n_seq > 65535) return dfail(TSB_ERR_UNSUPPORTED, "gated_delta: at most 65535 heads and sequences");
    return TSB_OK;
}
int64_t max_chunks(const tsb_delta_desc* d) {
    return std::min<int64_t>(d->n_tok / kChunk + d->n_seq, (int64_t) d->n_seq * ((d->max_len + kChunk - 1) / kChunk));
}
int64_t chunk_bytes(const tsb_delta_desc* d) {
    const int a = d->k_heads, b = d->v_heads;
    const bool half = d->dim_k == 64;
    if (d->elem_type == E_F32) return half ? Tiles<E_F32, 64>::chunk_bytes(a, b) : Tiles<E_F32, 128>::chunk_bytes(a, b);
    if (d->elem_type == E_F16) return half ? Tiles<E_F16, 64>::chunk_bytes(a, b) : Tiles<E_F16, 128>::chunk_bytes(a, b);
    return half ? Tiles<E_BF16, 64>::chunk_bytes(a, b) : Tiles<E_BF16, 128>::chunk_bytes(a, b);
}

template <int E, int DK, int W>
int launch_scan(const DeltaParams& p, cudaStream_t st) {
    constexpr int un = W == 1 ? 8 : 2;
    constexpr int sm = 2 * Tiles<E, DK>::kStage + (W == 1 ? 0 : un * 12 * 1024);
    static_assert(sm <= 226 * 1024, "shared memory");
    if (cudaFuncSetAttribute(k_delta_scan<E, DK, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) != cudaSuccess)
        return dcuda("gated_delta: shared memory");
    k_delta_scan<E, DK, W><<<dim3((unsigned) ((p.dv + 16 * un - 1) / (16 * un)), p.hv, p.n_seq), 256, sm, st>>>(p);
    return dcuda("gated_delta");
}
template <int E, int DK>
int launch_chunks(const DeltaParams& p, cudaStream_t st) {
    using T = Tiles<E, DK>;
    constexpr int sm = (T::kVal > T::kHead ? T::kVal : T::kHead) + (64 * LA + 32 * 36) * 4;
    if (cudaFuncSetAttribute(k_delta_prepare<E, DK>, cudaFuncAttributeMaxDynamicSharedMemorySize, sm) != cudaSuccess)
        return dcuda("gated_delta: shared memory");
    k_delta_prepare<E, DK><<<dim3((unsigned) p.max_chunks, p.hk), 128, sm, st>>>(p);
    if (int rc = dcuda("gated_delta: chunks")) return rc;
    // W 1 does less in all and W 2 a chunk sooner, so W 1 where the chunks of all sequences outweigh the longest one's, and where its
    // eight units a CTA have 16 columns each.  Measured with 32 heads of 128 (us a pass, W 1 against W 2): one sequence of 8192
    // tokens 1221 against 466, 8 ragged ones up to 1024 234 against 170 (fp32); 4 of 1000 226 against 249 (fp32 286 against 323), 16
    // of 256 248 against 272, 64 of 64 290 against 431; 16 of 256 with 6 heads 78 against 78; with heads of 64 143 against 128.
    const int64_t longest = (p.max_len + kChunk - 1) / kChunk;
    const bool many = p.dv > 64 && (int64_t) p.max_chunks * p.hv * 5 >= longest * sm_count() * 3;
    return many ? launch_scan<E, DK, 1>(p, st) : launch_scan<E, DK, 2>(p, st);
}
template <int DK>
int launch_type(const DeltaParams& p, cudaStream_t st) {
    return p.type == E_F32 ? launch_chunks<E_F32, DK>(p, st) : p.type == E_F16 ? launch_chunks<E_F16, DK>(p, st) : launch_chunks<E_BF16, DK>(p, st);
}

}  // namespace

// This file's copy of the bound of the waits (tsb_set_wait_limit_ns writes each).
int delta_set_wait_limit(unsigned long long ns) {
    return cudaMemcpyToSymbol(g_wait_ns, &ns, sizeof ns) == cudaSuccess ? TSB_OK : TSB_ERR_CUDA;
}

}  // namespace tsb

using namespace tsb;

extern "C" {

uint64_t tsb_gated_delta_workspace_bytes(const tsb_delta_desc* d) {
    if (delta_check(d) != TSB_OK || d->max_len <= kStepTokens) return 0;
    return (uint64_t) (max_chunks(d) * chunk_bytes(d));
}

int tsb_gated_delta(const tsb_delta_desc* d, const void* q, const void* k, const void* v, const float* g, const float* beta,
                    const float* state_in, float* state_out, const int32_t* state_idx, const int32_t* cu_seqlens, void* o,
                    void* workspace, uint64_t ws_bytes, void* stream) {
    if (int rc = delta_check(d)) return rc;
    if (d->n_seq == 0) return TSB_OK;
    if (d->n_tok && (!q || !k || !v || !g || !beta || !o)) return dfail(TSB_ERR_ARG, "gated_delta: null pointer");
    if (d->n_states && (!state_in || !state_out)) return dfail(TSB_ERR_ARG, "gated_delta: null state");
    if (!cu_seqlens && d->n_tok < (int64_t) d->n_seq * d->max_len)
        return dfail(TSB_ERR_ARG, "gated_delta: without cu_seqlens every sequence has max_len tokens");
    const int es = elem_bytes(d->elem_type);
    if ((uintptr_t) q % es || (uintptr_t) k % es || (uintptr_t) v % es || (uintptr_t) o % es || (uintptr_t) state_in % 16 ||
        (uintptr_t) state_out % 16)
        return dfail(TSB_ERR_ALIGN, "gated_delta: element alignment, states on 16 bytes");
    DeltaParams p{};
    p.q = q, p.k = k, p.v = v, p.g = g, p.beta = beta, p.s_in = state_in, p.s_out = state_out, p.idx = state_idx, p.cu = cu_seqlens;
    p.o = o, p.type = d->elem_type, p.n_seq = d->n_seq, p.max_len = d->max_len, p.hk = d->k_heads, p.hv = d->v_heads;
    p.dk = d->dim_k, p.dv = d->dim_v, p.n_states = d->n_states, p.n_tok = d->n_tok;
    p.q_tok = d->q_tok, p.q_head = d->q_head, p.k_tok = d->k_tok, p.k_head = d->k_head;
    p.v_tok = d->v_tok, p.v_head = d->v_head, p.o_tok = d->o_tok, p.o_head = d->o_head, p.gb_tok = d->gb_tok;
    p.scale = d->scale, p.eps = d->eps, p.norm = d->qk_norm != 0;
    p.wide = !((uintptr_t) q % 16 || (uintptr_t) k % 16 || (p.q_tok * es) % 16 || (p.q_head * es) % 16 || (p.k_tok * es) % 16 ||
               (p.k_head * es) % 16);
    p.err = device_error_word();
    cudaStream_t st = (cudaStream_t) stream;
    if (d->max_len <= kStepTokens) {
        const dim3 grid((d->dim_v + 31) / 32, d->v_heads, d->n_seq);
        if (d->dim_k == 64) k_delta_step<64><<<grid, 256, 0, st>>>(p);
        else k_delta_step<128><<<grid, 256, 0, st>>>(p);
        return dcuda("gated_delta");
    }
    const uint64_t need = tsb_gated_delta_workspace_bytes(d);
    if (!workspace || ws_bytes < need)
        return dfail(TSB_ERR_WORKSPACE, "gated_delta: workspace of %llu bytes needed", (unsigned long long) need);
    if ((uintptr_t) workspace % 16) return dfail(TSB_ERR_ALIGN, "gated_delta: 16-byte aligned workspace");
    if (max_chunks(d) > 0x7fffffffll) return dfail(TSB_ERR_UNSUPPORTED, "gated_delta: too many tokens");
    p.ws = (uint8_t*) workspace;
    p.max_chunks = (int) max_chunks(d);
    return d->dim_k == 64 ? launch_type<64>(p, st) : launch_type<128>(p, st);
}

}  // extern "C"
