// Serving many sequences from a paged KV cache: appending rotated keys and
// values, attention of the new tokens over the cache, sampling.  Ordinary
// floating point, no LNS: the ops a host runs outside LNS.  The code does not
// depend on the summation mode; every library of the build carries it.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include "lnsb200.h"
#include "lnsb_launch.cuh"

namespace cg = cooperative_groups;

namespace lnsb {
namespace {

// page ids outside the cache, waits that ran out: lnsb_paged_errors
__device__ unsigned long long g_paged_errors[2];

constexpr int k_sms = 148;                      // of one B200

template <class T> struct num;
template <> struct num<float> {
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct num<__half> {
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
    static constexpr uint32_t one2 = 0x3C003C00u;
    static constexpr float head = 7.0f;         // the largest weight is 2^7 at least, where its reference is set
};
template <> struct num<__nv_bfloat16> {
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xFFFF0000u));
    }
    static constexpr uint32_t one2 = 0x3F803F80u;
    static constexpr float head = 0.0f;
};

// two floats in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 c;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 z, x, y;\nmov.b64 {%0, %1}, z;\n}\n"
        : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 c;
    asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 z, x, y;\nmov.b64 {%0, %1}, z;\n}\n"
        : "=f"(c.x), "=f"(c.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return c;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n.reg .b64 x, y, z, w;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
        "fma.rn.f32x2 w, x, y, z;\nmov.b64 {%0, %1}, w;\n}\n"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// ============================ the plan =====================================

// the device's view of lnsb_paged_kv
struct paged {
    const int32_t * table;
    const int32_t * q_start;
    const int32_t * kv_len;
    int64_t         table_ld, n_pages, n_tokens, max_kv;
    int64_t         page_stride, row_stride, head_stride;
    int             n_seqs, page_shift, n_head_kv;
};

struct seq_span {
    int64_t first, n, kv;      // first new token, how many, visible rows
};
__device__ __forceinline__ seq_span span_of(const paged & P, int s) {
    const int64_t a = min(max((int64_t) P.q_start[s], (int64_t) 0), P.n_tokens);
    const int64_t b = min(max((int64_t) P.q_start[s + 1], a), P.n_tokens);
    return { a, b - a, min(max((int64_t) P.kv_len[s], (int64_t) 0), P.max_kv) };
}
// page id of a row below kv_len, or -1 (counted) for one outside the cache
__device__ __forceinline__ int64_t page_of(const paged & P, int s, int64_t row, bool count = true) {
    const int64_t id = P.table[s * P.table_ld + (row >> P.page_shift)];
    if (id >= 0 && id < P.n_pages) return id;
    if (count) atomicAdd(&g_paged_errors[0], 1ull);
    return -1;
}

// ============================ append =======================================

// Any alignment and any n_dims: one thread a rotated pair, copied element or v
// element.  Each looks its token up for itself, and nothing is loaded wide: 333
// us where the kernel below takes 56.  It is there for rows that do not allow
// that one's 16-byte accesses; a decoder's do.
template <class TI, class TC>
__global__ void k_paged_append(paged P, const TI * __restrict__ k, const TI * __restrict__ v, const TI * __restrict__ q,
                               TC * __restrict__ q_out, const float * __restrict__ cos_sin, int64_t k_ld, int64_t v_ld,
                               int64_t q_ld, int64_t q_out_ld, int n_head, int D, int n_dims, int neox,
                               TC * __restrict__ kc, TC * __restrict__ vc) {
    pdl_entry();
    const int half = n_dims / 2, per = half + (D - n_dims);
    const int64_t row_work = (int64_t) (n_head + P.n_head_kv) * per + (int64_t) P.n_head_kv * D;
    const int64_t n = P.n_tokens * row_work;
    for (int64_t i = (int64_t) blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t) blockDim.x * gridDim.x) {
        const int64_t t = i / row_work;
        int64_t r = i - t * row_work;
        int lo = 0, hi = P.n_seqs;                       // the last sequence that starts at or before t
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (P.q_start[mid] <= t) lo = mid; else hi = mid;
        }
        const seq_span S = span_of(P, lo);
        const int64_t row = S.kv - S.n + (t - S.first);
        if (t < S.first || t >= S.first + S.n || row < 0) continue;
        const int64_t heads = n_head + P.n_head_kv;
        const bool is_v = r >= heads * per;
        const int64_t h = is_v ? (r - heads * per) / D : r / per;
        const bool to_cache = is_v || h >= n_head;
        int64_t at = 0;
        if (to_cache) {
            const int64_t id = page_of(P, lo, row, r == n_head * per);      // counted by the token's first key element
            if (id < 0) continue;
            at = id * P.page_stride + (row & ((1 << P.page_shift) - 1)) * P.row_stride +
                 (is_v ? h : h - n_head) * P.head_stride;
        }
        if (is_v) {
            const int64_t d = (r - heads * per) % D;
            vc[at + d] = num<TC>::from(num<TI>::to(v[t * v_ld + h * D + d]));
            continue;
        }
        const int j = (int) (r - h * per);
        const TI * src = h < n_head ? q + t * q_ld + h * D : k + t * k_ld + (h - n_head) * D;
        TC * dst = h < n_head ? q_out + t * q_out_ld + h * D : kc + at;
        if (j >= half) {
            const int d = n_dims + j - half;
            dst[d] = num<TC>::from(num<TI>::to(src[d]));
            continue;
        }
        const int d0 = neox ? j : 2 * j, d1 = neox ? j + half : 2 * j + 1;
        const float c = cos_sin[(row * half + j) * 2], s = cos_sin[(row * half + j) * 2 + 1];
        const float x0 = num<TI>::to(src[d0]), x1 = num<TI>::to(src[d1]);
        dst[d0] = num<TC>::from(x0 * c - x1 * s);
        dst[d1] = num<TC>::from(x0 * s + x1 * c);
    }
}

// 8 elements at a 16-byte boundary
template <class T>
__device__ __forceinline__ void load8(const T * p, float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
        x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
        const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p));
        const uint32_t w[4] = { v.x, v.y, v.z, v.w };
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint16_t h = (uint16_t) (w[i / 2] >> (16 * (i & 1)));
            x[i] = num<T>::to(*reinterpret_cast<const T *>(&h));
        }
    }
}
template <class T>
__device__ __forceinline__ void store8(T * p, const float (&x)[8]) {
    *reinterpret_cast<uint4 *>(p) = make_uint4(num<T>::pack(x[0], x[1]), num<T>::pack(x[2], x[3]), num<T>::pack(x[4], x[5]),
                                               num<T>::pack(x[6], x[7]));
}

// Where rows lie at 16-byte boundaries and n_dims is a multiple of 16: a thread
// takes 8 elements (NEOX: 8 of each half of the pairs), a block `tokens`
// tokens.  Its inputs are on their way while the first threads look up where
// the block's tokens go.  HBM bounds it: 8,592 tokens of 32/8 heads of 128 from
// F32 56 us, 5.7 TB/s (the element-wise kernel 333 us); one token 2.2 us.
template <class TI, class TC, bool NEOX>
__global__ void __launch_bounds__(256)
k_paged_append_vec(paged P, const TI * __restrict__ k, const TI * __restrict__ v, const TI * __restrict__ q,
                   TC * __restrict__ q_out, const float * __restrict__ cos_sin, int64_t k_ld, int64_t v_ld, int64_t q_ld,
                   int64_t q_out_ld, int n_head, int D, int n_dims, int tokens, TC * __restrict__ kc, TC * __restrict__ vc) {
    __shared__ int64_t s_at[256];                       // the token's place in a head of the caches, -1: none
    __shared__ int     s_row[256];                      // its row, negative: none
    pdl_entry();
    const int tid = threadIdx.x, half = n_dims / 2;
    const int turned = NEOX ? half / 8 : n_dims / 8;    // units of a q or k head: turned ones, then copied ones
    const int per = turned + (D - n_dims) / 8, qk = (n_head + P.n_head_kv) * per, units = qk + P.n_head_kv * (D / 8);
    const int64_t t0 = (int64_t) blockIdx.x * tokens;
    bool planned = false;
    for (int i = tid; i - tid < tokens * units; i += 256) {
        const bool in = i < tokens * units;
        const int tb = tokens == 1 ? 0 : i / units, r = i - tb * units;
        const int64_t t = t0 + tb;
        const bool live = in && t < P.n_tokens, is_v = r >= qk;
        const int h = is_v ? (r - qk) / (D / 8) : r / per, j = is_v ? (r - qk) % (D / 8) : r % per;
        const bool is_q = !is_v && h < n_head, turn = !is_v && j < turned;
        const int kvh = is_v ? h : h - n_head;
        // NEOX: dims 8 j and half + 8 j of the pairs, copied units after both halves
        const int d = turn || is_v ? 8 * j : n_dims + 8 * (j - turned);
        float x[8], y[8];
        if (live) {
            const TI * src = (is_q ? q + t * q_ld + (int64_t) h * D : is_v ? v + t * v_ld + (int64_t) kvh * D
                                                                           : k + t * k_ld + (int64_t) kvh * D) + d;
            load8(src, x);
            if (NEOX && turn) load8(src + half, y);
        }
        if (!planned) {
            planned = true;
            if (tid < tokens) {
                const int64_t tt = t0 + tid;
                int row = -1;
                int64_t at = -1;
                if (tt < P.n_tokens) {
                    int lo = 0, hi = P.n_seqs;          // the last sequence that starts at or before the token
                    while (hi - lo > 1) {
                        const int mid = (lo + hi) / 2;
                        if (P.q_start[mid] <= tt) lo = mid; else hi = mid;
                    }
                    const seq_span S = span_of(P, lo);
                    const int64_t rw = S.kv - S.n + (tt - S.first);
                    if (tt >= S.first && tt < S.first + S.n && rw >= 0) {
                        row = (int) rw;
                        const int64_t id = page_of(P, lo, rw);
                        if (id >= 0) at = id * P.page_stride + (rw & ((1 << P.page_shift) - 1)) * P.row_stride;
                    }
                }
                s_row[tid] = row;
                s_at[tid] = at;
            }
            __syncthreads();
        }
        if (!live) continue;
        const int row = s_row[tb];
        const int64_t at = s_at[tb];
        if (row < 0 || (!is_q && at < 0)) continue;
        TC * dst = (is_q ? q_out + t * q_out_ld + (int64_t) h * D : (is_v ? vc : kc) + at + kvh * P.head_stride) + d;
        if (turn) {
            float c[8], s[8];
            const float4 * cs = reinterpret_cast<const float4 *>(cos_sin + ((int64_t) row * half + (NEOX ? 8 : 4) * j) * 2);
#pragma unroll
            for (int e = 0; e < (NEOX ? 4 : 2); e++) {
                const float4 w = __ldg(cs + e);
                c[2 * e] = w.x, s[2 * e] = w.y, c[2 * e + 1] = w.z, s[2 * e + 1] = w.w;
            }
            if (NEOX) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float a = x[e], b = y[e];
                    x[e] = a * c[e] - b * s[e];
                    y[e] = a * s[e] + b * c[e];
                }
                store8(dst + half, y);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float a = x[2 * e], b = x[2 * e + 1];
                    x[2 * e] = a * c[e] - b * s[e];
                    x[2 * e + 1] = a * s[e] + b * c[e];
                }
            }
        }
        store8(dst, x);
    }
}

// ===================== attention: few rows a sequence ======================
//
// The rows of one (sequence, kv head) are its (token, head of the group)
// pairs, row r = token r / G, head r % G.  A CTA takes 16 of them -- the
// height of one mma.sync tile -- over a range of 64-key tiles: warp w
// computes keys 16 w .. 16 w + 15 of each tile, with its own maximum, sum and
// output, so the four warps never wait for one another inside the range and
// join at its end.
//
// What bounds it is the cache's bytes.  All (sequence, row tile, kv head, key
// tile) units form one line that the CTAs cut into equal shares, whatever the
// lengths: a share that ends inside an item leaves a partial result in `work`,
// and the CTA that comes last to an item joins its partials in the order of
// the line, so the result does not hang on who came when.
//
// The maximum is a reference that moves only when a score passes it by more
// than 8 (in log2; the difference of near floats is exact, a sum with 8 need
// not be): exp2 of the rest stays below 2^8, and the quotient does not see the
// reference.  Half's numbers end at 2^-24, where BF16's go on: there it is 7
// below the score that sets it, so that weights down to 2^-32 of the largest
// count, and none passes 2^15.  The sum of the weights comes
// from the same product as the output, against a column of ones, so it is of
// the weights as rounded.
//
// The weights are rounded to the cache's type because the tensor cores take
// operands of one 16-bit type; two parts of each would double the products with
// V.  Against 64 bits the outputs are off by 2.1e-3 in BF16 and 2.3e-4 in F16
// (root mean square, relative), where rounding the outputs alone gives 1.7e-3
// and 2.2e-4.
//
// Measured, replayed from a CUDA graph: 64 ragged sequences of up to 8,192 rows,
// 32/8 heads of 128 (1.2 GB) 205 us, 5.9 TB/s; one token over 131,072 rows 109
// us, 4.9 TB/s; one token over 200 rows 8.3 us.

constexpr int ROWS = 16, KEYS = 64, A_CTAS = 2 * k_sms;
constexpr int MAX_DIM = 256;
constexpr float k_lag = 8.0f;
constexpr float k_none = -FLT_MAX;             // the reference of a row that has seen nothing

// work: [counters A_CTAS int32][partials A_CTAS * 2 * (ROWS * MAX_DIM + 2 * ROWS) float]
constexpr int64_t A_PART = ROWS * MAX_DIM + 2 * ROWS;
constexpr int64_t A_COUNT_BYTES = (A_CTAS * 4 + 255) / 256 * 256;
constexpr int64_t A_WORK = A_COUNT_BYTES + ((int64_t) A_CTAS * 2 * A_PART * 4 + 255) / 256 * 256;

__device__ __forceinline__ uint32_t smem_addr(const void * p) { return (uint32_t) __cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void * src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" :: "r"(dst), "l"(src), "r"(valid ? 16 : 0));
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;\n" :: "n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
template <class T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <class T>
__device__ __forceinline__ uint32_t pack2(uint32_t lo, uint32_t hi) {
    return num<T>::pack(__uint_as_float(lo), __uint_as_float(hi));
}

// units of one sequence in the line: row tiles x kv heads x key tiles
struct seq_units {
    int64_t row_tiles, key_tiles, first_tile;   // key tiles from first_tile on
};
__device__ __forceinline__ seq_units units_of(const seq_span & S, int G, int64_t window, int64_t rows_most) {
    seq_units u;
    u.row_tiles = S.n * G > rows_most ? 0 : (S.n * G + ROWS - 1) / ROWS;
    int64_t lo = 0;
    if (window > 0) lo = max((int64_t) 0, S.kv - S.n - window + 1);
    u.first_tile = lo / KEYS;
    u.key_tiles = max((int64_t) 1, (S.kv + KEYS - 1) / KEYS - u.first_tile);
    return u;
}
// smem of one CTA: the warps' rings, reused for joining the warps
template <int D> __host__ __device__ constexpr int a_stages() { return D <= 128 ? 3 : 2; }
template <int D> __host__ __device__ constexpr int a_stage_bytes() { return 16 * D * 2 * 2; }
template <int D> __host__ __device__ constexpr int a_smem() {
    const int ring = 4 * a_stages<D>() * a_stage_bytes<D>();
    const int join = 4 * (ROWS * (D + 4) + 2 * ROWS) * 4;
    return ring > join ? ring : join;
}
// 16-byte chunk c of row r in a [rows][D] tile: the rows that one ldmatrix
// reads together lie in different banks
template <int D> __device__ __forceinline__ uint32_t chunk_at(int r, int c) {
    constexpr int CPR = D / 8;
    const int x = CPR >= 8 ? (r & 7) : CPR == 4 ? ((r >> 1) & 3) : ((r >> 2) & 1);
    return (uint32_t) (r * CPR + (c ^ x)) * 16;
}

template <class T, int D>
__global__ void __launch_bounds__(128)
k_paged_attn_rows(paged P, const T * __restrict__ q, T * __restrict__ dst, const T * __restrict__ kc,
                  const T * __restrict__ vc, int64_t q_ld, int64_t dst_ld, int G, float scale_log2, int64_t window,
                  int64_t rows_most, int * __restrict__ counters, float * __restrict__ parts) {
    constexpr int ST = a_stages<D>(), SB = a_stage_bytes<D>(), CPR = D / 8, KS = D / 16;
    constexpr float head = num<T>::head, lag = k_lag + head;
    extern __shared__ __align__(128) unsigned char sm[];
    __shared__ int64_t s_scan[128];
    __shared__ int s_last;
    pdl_entry();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int c = blockIdx.x;

    // the line's length: thread t sums the sequences of its share
    const int per = (P.n_seqs + 127) / 128;
    const int s_lo = min(tid * per, P.n_seqs), s_hi = min(s_lo + per, P.n_seqs);
    int64_t mine = 0;
    for (int s = s_lo; s < s_hi; s++) {
        const seq_units u = units_of(span_of(P, s), G, window, rows_most);
        mine += u.row_tiles * u.key_tiles * P.n_head_kv;
    }
    s_scan[tid] = mine;
    __syncthreads();
    int64_t W = 0;
    for (int i = 0; i < 128; i++) W += s_scan[i];
    const int64_t N = min((int64_t) gridDim.x, W);                // CTAs that get a share: one unit at least
    if (c >= N) return;
    int64_t x = W * c / N;
    const int64_t x_end = W * (c + 1) / N;
    // the sequence that holds unit x, and the line's position where it begins
    int s = 0;
    int64_t base = 0;
    {
        int b = 0;
        while (base + s_scan[b] <= x) base += s_scan[b++];
        s = b * per;
    }
    const uint32_t ring = smem_addr(sm) + warp * ST * SB;
    float * join = reinterpret_cast<float *>(sm);

    while (x < x_end) {
        seq_span S = span_of(P, s);
        seq_units u = units_of(S, G, window, rows_most);
        int64_t len = u.row_tiles * u.key_tiles * P.n_head_kv;
        while (base + len <= x) {
            base += len;
            S = span_of(P, ++s);
            u = units_of(S, G, window, rows_most);
            len = u.row_tiles * u.key_tiles * P.n_head_kv;
        }
        const int64_t item = (x - base) / u.key_tiles;           // (row tile, kv head) of the sequence
        const int64_t item0 = base + item * u.key_tiles;         // its place on the line
        const int64_t t0 = x - item0, t1 = min(u.key_tiles, x_end - item0);
        const int h = (int) (item % P.n_head_kv);
        const int64_t r0 = item / P.n_head_kv * ROWS, R = S.n * G;
        const int64_t pos0 = S.kv - S.n;                         // row of the sequence's first new token
        // keys that some row of the tile sees
        const int64_t last_row = min(r0 + ROWS, R) - 1;
        const int64_t key_end = min(S.kv, pos0 + last_row / G + 1);
        const int64_t key_lo = window > 0 ? max((int64_t) 0, pos0 + r0 / G - window + 1) : 0;

        // rows lane/4 and lane/4 + 8 of the tile
        int64_t pos[2], lo[2];
        const T * qp[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int64_t r = r0 + lane / 4 + 8 * i;
            pos[i] = r < R ? pos0 + r / G : -1;
            lo[i] = window > 0 ? pos[i] - window + 1 : 0;
            qp[i] = r < R ? q + (S.first + r / G) * q_ld + ((int64_t) h * G + r % G) * D + (lane % 4) * 2 : nullptr;
        }
        uint32_t qf[KS][4];
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                qf[k][i] = qp[i & 1] ? *reinterpret_cast<const uint32_t *>(qp[i & 1] + k * 16 + (i >> 1) * 8) : 0u;

        float o[D / 8][4], l[4] = { 0, 0, 0, 0 }, m[2] = { k_none, k_none };
#pragma unroll
        for (int i = 0; i < D / 8; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[i][e] = 0.0f;

        const T * kh = kc + (int64_t) h * P.head_stride;
        const T * vh = vc + (int64_t) h * P.head_stride;
        // the keys of tile t that this warp takes
        auto load = [&](int64_t t, int stage) {
            const int64_t k0 = (u.first_tile + t) * KEYS + warp * 16;
            const uint32_t ks = ring + stage * SB, vs = ks + 16 * D * 2;
            int64_t id[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {                        // page_size >= 8: eight keys share a page
                const int64_t key = k0 + 8 * i;
                id[i] = t < t1 && key < key_end && key + 8 > key_lo ? page_of(P, s, key) : -1;
            }
#pragma unroll
            for (int j = 0; j < 16 * CPR / 32; j++) {
                const int idx = j * 32 + lane, r = idx / CPR, ch = idx % CPR;
                const int64_t key = k0 + r, pid = id[r >> 3];
                const bool ok = pid >= 0 && key < key_end && key >= key_lo;
                const int64_t off = ok ? pid * P.page_stride + (key & ((1 << P.page_shift) - 1)) * P.row_stride + ch * 8 : 0;
                cp16(ks + chunk_at<D>(r, ch), kh + off, ok);
                cp16(vs + chunk_at<D>(r, ch), vh + off, ok);
            }
            cp_commit();
        };
        for (int i = 0; i < ST - 1; i++) load(t0 + i, i);
        int stage = 0;
        for (int64_t t = t0; t < t1; t++) {
            load(t + ST - 1, stage == 0 ? ST - 1 : stage - 1);
            cp_wait<ST - 1>();
            __syncwarp();
            const uint32_t ks = ring + stage * SB, vs = ks + 16 * D * 2;
            float sc[2][4] = {};
#pragma unroll
            for (int k = 0; k < KS; k++) {
                uint32_t b[4];                                    // keys 0-7 and 8-15, halves of 16 dims
                ldsm4(ks + chunk_at<D>((lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)), b);
                mma16816<T>(sc[0], qf[k], b[0], b[1]);
                mma16816<T>(sc[1], qf[k], b[2], b[3]);
            }
            const int64_t k0 = (u.first_tile + t) * KEYS + warp * 16;
            float top[2] = { -INFINITY, -INFINITY };
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int64_t key = k0 + n * 8 + (lane % 4) * 2 + (e & 1);
                    const int i = e >> 1;
                    sc[n][e] = key <= pos[i] && key >= lo[i] ? __fmul_rn(sc[n][e], scale_log2) : -INFINITY;
                    top[i] = fmaxf(top[i], sc[n][e]);
                }
            if (__any_sync(0xFFFFFFFFu, top[0] - m[0] > lag || top[1] - m[1] > lag)) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 1));
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xFFFFFFFFu, top[i], 2));
                    const float mn = fmaxf(m[i], top[i] - head), f = ex2(m[i] - mn);
                    m[i] = mn;
                    l[2 * i] *= f;
#pragma unroll
                    for (int d = 0; d < D / 8; d++) {
                        o[d][2 * i] *= f;
                        o[d][2 * i + 1] *= f;
                    }
                }
            }
            uint32_t p[4];
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int i = 0; i < 2; i++)
                    p[2 * n + i] = num<T>::pack(ex2(sc[n][2 * i] - m[i]), ex2(sc[n][2 * i + 1] - m[i]));
            mma16816<T>(l, p, num<T>::one2, num<T>::one2);
#pragma unroll
            for (int d = 0; d < D / 16; d++) {
                uint32_t b[4];
                ldsm4t(vs + chunk_at<D>((lane & 7) + (((lane >> 3) & 1) << 3), 2 * d + (lane >> 4)), b);
                mma16816<T>(o[2 * d], p, b[0], b[1]);
                mma16816<T>(o[2 * d + 1], p, b[2], b[3]);
            }
            __syncwarp();
            stage = stage + 1 == ST ? 0 : stage + 1;
        }
        cp_wait<0>();
        __syncthreads();

        // join the four warps: [warp][row][D + 4] outputs, then maxima and sums
        float * jm = join + 4 * ROWS * (D + 4), * jl = jm + 4 * ROWS;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = lane / 4 + 8 * i;
            if (lane % 4 == 0) {
                jm[warp * ROWS + r] = m[i];
                jl[warp * ROWS + r] = l[2 * i];
            }
#pragma unroll
            for (int d = 0; d < D / 8; d++)
                *reinterpret_cast<float2 *>(join + (warp * ROWS + r) * (D + 4) + d * 8 + (lane % 4) * 2) =
                    make_float2(o[d][2 * i], o[d][2 * i + 1]);
        }
        __syncthreads();
        const int rows = (int) min((int64_t) ROWS, R - r0);
        const bool whole = t0 == 0 && t1 == u.key_tiles;
        float * part = parts + ((int64_t) c * 2 + (t0 == 0)) * A_PART;   // an item that began here, or before
        for (int i = tid; i < rows * D; i += 128) {
            const int r = i / D, d = i % D;
            float mx = jm[r];
#pragma unroll
            for (int w = 1; w < 4; w++) mx = fmaxf(mx, jm[w * ROWS + r]);
            float num_ = 0, den = 0;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = ex2(jm[w * ROWS + r] - mx);
                num_ += f * join[(w * ROWS + r) * (D + 4) + d];
                den += f * jl[w * ROWS + r];
            }
            if (whole) {
                const int64_t gr = r0 + r;
                dst[(S.first + gr / G) * dst_ld + ((int64_t) h * G + gr % G) * D + d] = num<T>::from(den != 0 ? num_ / den : 0.0f);
            } else {
                part[r * D + d] = num_;
                if (d == 0) {
                    part[ROWS * MAX_DIM + r] = mx;
                    part[ROWS * MAX_DIM + ROWS + r] = den;
                }
            }
        }
        if (!whole) {
            // CTA b holds unit y where W b / N <= y: the ones that share the item
            const int64_t y1 = item0 + u.key_tiles - 1;
            const int c0 = (int) (((item0 + 1) * N - 1) / W), c1 = (int) (((y1 + 1) * N - 1) / W);
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicAdd(&counters[c0], 1) == c1 - c0;
            __syncthreads();
            if (s_last) {
                __threadfence();
                for (int i = tid; i < rows * D; i += 128) {
                    const int r = i / D, d = i % D;
                    float mx = k_none, num_ = 0, den = 0;
                    for (int b = c0; b <= c1; b++) {
                        const float * pb = parts + ((int64_t) b * 2 + (b == c0)) * A_PART;
                        const float mb = __ldcg(pb + ROWS * MAX_DIM + r), mn = fmaxf(mx, mb);
                        const float f = ex2(mx - mn), g = ex2(mb - mn);
                        num_ = num_ * f + g * __ldcg(pb + r * D + d);
                        den = den * f + g * __ldcg(pb + ROWS * MAX_DIM + ROWS + r);
                        mx = mn;
                    }
                    const int64_t gr = r0 + r;
                    dst[(S.first + gr / G) * dst_ld + ((int64_t) h * G + gr % G) * D + d] =
                        num<T>::from(den != 0 ? num_ / den : 0.0f);
                }
                if (tid == 0) counters[c0] = 0;
            }
        }
        __syncthreads();                                          // the ring is free again
        x = item0 + t1;
    }
}

// ===================== attention: chunks ===================================
//
// Sequences with more than 16 rows (token, head of the group) go to the
// tensor cores in tiles of 256 rows, two groups of 128, over tiles of keys.
// S = Q K^T of a group lands in TMEM, one row a lane; the group's 128 threads
// read one row each, so maximum and sum need no other thread, and write the
// weights back into the same columns as the 16-bit A operand of P V, whose sum
// O stays in TMEM.  They add up the weights as rounded, as the rows kernel does
// (sums of the weights in 32 bits are 1-2 % faster, and off by a heavy weight's
// rounding).
//
// Head dim 64 leaves TMEM for two S of 64 keys to each group: while its softmax
// works on one, the next is ready, so it waits for no product (45 us where one
// S of 128 keys took 57 when the two were compared, on 16 sequences of up to 512
// new tokens in a window of 1,024).  At 128 the products are what counts, and QK
// over 64 keys reads shared memory for Q as long as over 128: one S of 128 keys
// (720 us where two of 64 took 998, on the two chunks below), and PV of its first
// 64 keys starts under the weights of the others.
//
// Measured, replayed from a CUDA graph: two chunks, 3,927 tokens over 26,803 rows
// in all, 32/8 heads of 128, 734 us (1,087 TFLOP/s; 847 us call after call);
// 512 tokens over 8,192 rows 85 us; the 16 sequences 47 us, behind the rows
// kernel, whose CTAs leave no registers for this kernel's to start beside them.
//
//   warps 0-3, 4-7  group 0, group 1: Q into shared memory, softmax, output
//   warp 8          one thread issues every MMA: PV of a group's tile j, then
//                   its QK of the next tile for that S, one group after the
//                   other, so one group's softmax runs under the other's
//                   products
//   warp 9          TMA of K and V pages through a ring of tiles
//   warp 10         walks the CTA's share of the line and hands out its items
//   warp 11         nothing: it completes the warpgroup that gives registers to
//                   the softmax at head dim 128 (168 x 384 at launch = 208 x 256
//                   + 88 x 128)
//
// TMEM operations of one thread run in the order of their issue: QK of the
// next tile may overwrite the weights that PV of tile j reads.  As with few rows,
// the (row tile, kv head, key tile) units of all sequences form a line that
// the CTAs cut into equal shares; each warp joins its own 32 rows of a cut
// item, so no warp waits for another outside the mbarriers.
//
// Every wait gives up after a limit (lnsb_paged_attn_wait_limit): the CTA then
// drains what it has in flight, frees its TMEM and counts a timeout, for the
// device and in `work`.

constexpr int B_ROWS = 128, B_TILE = 256, B_THREADS = 384, B_SUMS = 256, B_ITEMS = 4, B_CTAS = k_sms;
constexpr uint32_t k_wait_cycles = 1u << 31;

// work, behind the rows kernel's: counters, partials, and the waits that ran out
// partials: [slot][group][warp][d / 4][lane] float4, then [warp][lane] (m, l)
constexpr int64_t B_PART = (int64_t) B_TILE * (128 + 2);
constexpr int64_t B_COUNT_BYTES = ((int64_t) B_CTAS * 8 * 4 + 255) / 256 * 256;
constexpr int64_t B_WORK = B_COUNT_BYTES + (int64_t) B_CTAS * 2 * B_PART * 4;
constexpr int64_t WORK_BYTES = A_WORK + B_WORK + 8;
static_assert(B_WORK % 8 == 0, "the count's place");

// ---- mbarriers, TMA, tcgen05 ----
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" :: "r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" :: "r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
struct give_up {
    int      stop;                   // a wait has run out
    uint32_t limit;                  // cycles
};
// false: the CTA gives up (this wait ran out, or another one did)
__device__ __forceinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile give_up * stop) {
    const uint32_t t0 = (uint32_t) clock();
    while (!bar_try(bar, parity)) {
        if (stop->stop) return false;
        if ((uint32_t) clock() - t0 > stop->limit) {
            stop->stop = 1;
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile give_up * stop) {
    return bar_try(bar, parity) || bar_wait_slow(bar, parity, stop);
}
// the same for a whole warp: all its lanes go on, or none
__device__ __forceinline__ bool bar_wait_warp(uint32_t bar, uint32_t parity, volatile give_up * stop) {
    return __all_sync(0xFFFFFFFFu, bar_wait(bar, parity, stop));
}
__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap * map, int d, int row, int head, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n"
                 :: "r"(dst), "l"(map), "r"(d), "r"(row), "r"(head), "r"(page), "r"(bar) : "memory");
}
// operand in shared memory, 128-byte swizzle: start, stride between the
// 64-element halves (major dimension outside), stride between groups of 8 rows
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    return (uint64_t) ((addr & 0x3FFFF) >> 4) | ((uint64_t) (lead >> 4) << 16) | ((uint64_t) (stride >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t) add) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t) add) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" :: "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
// the loads of v are complete; v is used only behind this
template <int N> __device__ __forceinline__ void tc_wait_ld(uint32_t (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(v[i]));
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
#define LNSB_R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
#define LNSB_W4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
// 32 columns of the warp's 32 lanes
__device__ __forceinline__ void tc_ld32(uint32_t a, uint32_t * v) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
                 "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : LNSB_R4(v, 0), LNSB_R4(v, 4), LNSB_R4(v, 8), LNSB_R4(v, 12), LNSB_R4(v, 16), LNSB_R4(v, 20), LNSB_R4(v, 24),
                   LNSB_R4(v, 28) : "r"(a));
}
__device__ __forceinline__ void tc_st32(uint32_t a, const uint32_t * v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
                 "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n"
                 :: "r"(a), LNSB_W4(v, 0), LNSB_W4(v, 4), LNSB_W4(v, 8), LNSB_W4(v, 12), LNSB_W4(v, 16), LNSB_W4(v, 20),
                    LNSB_W4(v, 24), LNSB_W4(v, 28) : "memory");
}
#undef LNSB_R4
#undef LNSB_W4

// ---- the line ----
struct tile_plan {
    int64_t rows_above, window;      // sequences of more rows than this
    int     G, key_shift;            // heads to a kv head; log2 of the keys of a tile
};
// key tiles [lo, hi) of row tile rt of a sequence; one at least
__device__ __forceinline__ void tile_keys(const tile_plan & L, const seq_span & S, int64_t rt, int64_t & lo, int64_t & n) {
    const int64_t pos0 = S.kv - S.n;
    const uint32_t R = (uint32_t) (S.n * L.G), r0 = (uint32_t) rt * B_TILE;      // below 2^31
    const uint32_t last = (min(r0 + B_TILE, R) - 1) / (uint32_t) L.G, first = r0 / (uint32_t) L.G;
    const int64_t hi = (max(min(S.kv, pos0 + last + 1), (int64_t) 0) + (1 << L.key_shift) - 1) >> L.key_shift;
    lo = L.window > 0 ? max((int64_t) 0, pos0 + first - L.window + 1) >> L.key_shift : 0;
    n = max((int64_t) 1, hi - lo);
}
__device__ __forceinline__ int64_t row_tiles_of(const tile_plan & L, const seq_span & S) {
    const int64_t R = S.n * L.G;
    return R > L.rows_above ? (R + B_TILE - 1) / B_TILE : 0;
}
// units of one kv head of a sequence, summed by the whole warp
__device__ __forceinline__ int64_t units_by_warp(const tile_plan & L, const seq_span & S) {
    const int64_t nr = row_tiles_of(L, S);
    int64_t sum = 0;
    for (int64_t rt = threadIdx.x & 31; rt < nr; rt += 32) {
        int64_t lo, n;
        tile_keys(L, S, rt, lo, n);
        sum += n;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
    return sum;
}
// a CTA's part of one item
struct tile_item {
    int seq, head;                   // kv head
    int first, kv, pos0;             // the sequence's first new token, its cached rows, cache row of the first new token
    int r0, rows;                    // first row of the tile; all rows of the sequence
    int key0, n;                     // first key, and how many key tiles (0: the share is done)
    int cut, c0, others;             // part of an item that others share: their first CTA, and how many more there are
};
// walks the CTA's share [x, x_end) of the line; the whole warp takes part
struct line_walk {
    const int64_t * sums;            // units of each run of `per` sequences
    int64_t per, W, N, x, x_end, base, run_base, seq_len;   // seq_len: units of sequence s, from base on
    int     run, s;

    __device__ void next(const paged & P, const tile_plan & L, tile_item & I) {
        I.n = 0;
        if (x >= x_end) return;
        const int lane = threadIdx.x & 31;
        // the run of sequences, then the sequence, that holds unit x
        bool moved = seq_len < 0;
        while (run_base + sums[run] <= x) {
            run_base += sums[run++];
            moved = true;
        }
        if (moved) {
            s = (int) (run * per);
            base = run_base;
            seq_len = units_by_warp(L, span_of(P, s)) * P.n_head_kv;
        }
        while (base + seq_len <= x) {
            base += seq_len;
            seq_len = units_by_warp(L, span_of(P, ++s)) * P.n_head_kv;
        }
        const int64_t per_head = seq_len / P.n_head_kv;
        const seq_span S = span_of(P, s);
        I.seq = s;
        I.head = (int) ((x - base) / per_head);
        int64_t at = base + I.head * per_head, len = 1, lo0 = 0;   // the row tile's place on the line, its key tiles
        const int64_t nr = row_tiles_of(L, S);
        int64_t rt = 0;
        for (int64_t r = 0; r < nr; r += 32) {
            int64_t lo = 0, n = 0;
            if (r + lane < nr) tile_keys(L, S, r + lane, lo, n);
            int64_t upto = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
                if (lane >= d) upto += o;
            }
            const uint32_t hit = __ballot_sync(0xFFFFFFFFu, r + lane < nr && at + upto > x);
            if (hit) {
                const int l = __ffs(hit) - 1;
                rt = r + l;
                lo0 = __shfl_sync(0xFFFFFFFFu, lo, l);
                len = __shfl_sync(0xFFFFFFFFu, n, l);
                at += __shfl_sync(0xFFFFFFFFu, upto, l) - len;
                break;
            }
            at += __shfl_sync(0xFFFFFFFFu, upto, 31);
        }
        const int64_t t0 = x - at, t1 = min(len, x_end - at);
        I.first = (int) S.first;
        I.kv = (int) S.kv;
        I.pos0 = (int) (S.kv - S.n);
        I.r0 = (int) (rt * B_TILE);
        I.rows = (int) (S.n * L.G);
        I.key0 = (int) ((lo0 + t0) << L.key_shift);
        I.n = (int) (t1 - t0);
        I.cut = t0 > 0 || t1 < len;
        // CTA b holds unit y where W b / N <= y
        I.c0 = (int) (((at + 1) * N - 1) / W);
        I.others = (int) (((at + len) * N - 1) / W) - I.c0;
        x = at + t1;
    }
};

// the first cache row that the sequence still owns: the window's of its first new token
__device__ __forceinline__ int first_owned(const tile_item & I, const tile_plan & L) {
    return L.window > 0 ? (int) max((int64_t) 0, I.pos0 - L.window + 1) : 0;
}

// shared memory of one CTA
template <int D> __host__ __device__ constexpr int b_keys() { return D == 128 ? 128 : 64; }
template <int D> __host__ __device__ constexpr int b_tile_bytes() { return b_keys<D>() * D * 2; }
template <int D> __host__ __device__ constexpr int b_q_bytes() { return B_ROWS * D * 2; }
template <int D> __host__ __device__ constexpr int b_ring() { return D == 128 ? 5 : 10; }
struct tile_control {                // behind the tiles
    int64_t   sums[B_SUMS];
    tile_item item[B_ITEMS];
    uint64_t  bar[2 * 10 + 2 * B_ITEMS + 15];
    give_up   stop;
    uint32_t  tmem;
};
template <int D> __host__ __device__ constexpr int b_smem() {
    return 2 * b_q_bytes<D>() + b_ring<D>() * b_tile_bytes<D>() + (int) sizeof(tile_control);
}
static_assert(b_smem<128>() <= 227 * 1024 && b_smem<64>() <= 227 * 1024, "shared memory of one CTA");

template <class T, int D>
__global__ void __launch_bounds__(B_THREADS, 1)
k_paged_attn_tiles(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, paged P, tile_plan L,
                   const T * __restrict__ q, T * __restrict__ dst, int64_t q_ld, int64_t dst_ld, float scale_log2,
                   int * __restrict__ counters, float * __restrict__ parts, uint32_t wait_cycles, unsigned long long * __restrict__ ran_out) {
    // bytes of a K or V tile, of its 64-dim halves, and of Q's
    constexpr int B_KEYS = b_keys<D>(), BUFS = D == 128 ? 1 : 2, PARTS = B_KEYS / 64;
    constexpr int ST = b_ring<D>(), TB = b_tile_bytes<D>(), HB = B_KEYS * 128, QB = b_q_bytes<D>(), QH = B_ROWS * 128, HALVES = D / 64;
    constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
    constexpr float head = num<T>::head, lag = k_lag + head;
    // f32 sums of 16-bit operands, 128 rows; B of PV is [key][dim], keys outside
    constexpr uint32_t fmt = (1u << 4) | ((BF ? 1u : 0u) << 7) | ((BF ? 1u : 0u) << 10) | (8u << 24);
    constexpr uint32_t idesc_qk = fmt | ((B_KEYS / 8) << 17), idesc_pv = fmt | (1u << 16) | ((D / 8) << 17);
    constexpr uint32_t S_COL = 0, O_COL = 256;              // + 128 g (+ 64 for every other tile of 64 keys), + D g

    extern __shared__ __align__(1024) unsigned char tile_sm[];     // swizzled tiles: 1024-byte boundaries
    tile_control & C = *reinterpret_cast<tile_control *>(tile_sm + 2 * QB + ST * TB);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t q_sm = smem_addr(tile_sm), ring = q_sm + 2 * QB;
    const uint32_t bars = smem_addr(C.bar);
    const uint32_t kv_full = bars, kv_empty = bars + 8 * ST, q_full = kv_empty + 8 * ST, s_full = q_full + 16,
                   p_ready = s_full + 32, o_full = p_ready + 32, pv_done = o_full + 16, it_full = pv_done + 16, it_empty = it_full + 8 * B_ITEMS, drained = it_empty + 8 * B_ITEMS;
    volatile give_up * stop = &C.stop;

    if (tid == 0) {
        for (int i = 0; i < ST; i++) {
            bar_init(kv_full + 8 * i, 1);
            bar_init(kv_empty + 8 * i, 1);
        }
        for (int g = 0; g < 2; g++) {
            bar_init(q_full + 8 * g, B_ROWS);
            for (int b = 0; b < 2; b++) {
                bar_init(s_full + 16 * g + 8 * b, 1);
                bar_init(p_ready + 16 * g + 8 * b, B_ROWS);
            }
            bar_init(pv_done + 8 * g, 1);
            bar_init(o_full + 8 * g, 1);
        }
        for (int i = 0; i < B_ITEMS; i++) {
            bar_init(it_full + 8 * i, 1);
            bar_init(it_empty + 8 * i, 10);                  // warps 0 .. 9
        }
        bar_init(drained, 1);
        C.stop.limit = wait_cycles;
        C.stop.stop = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    // behind k_paged_attn_rows of the same call too: only a grid's own wait makes
    // visible to it what earlier grids wrote (q, the plan, the cache's rows)
    pdl_entry();

    // the line's length
    const int64_t per = (P.n_seqs + B_SUMS - 1) / B_SUMS;
    int64_t mine = 0;
    for (int64_t j = 0; j < (tid < B_SUMS ? per : 0); j++) {
        const int64_t s = tid * per + j;
        seq_span S = { 0, 0, 0 };
        if (s < P.n_seqs) S = span_of(P, (int) s);
        const int64_t nr = row_tiles_of(L, S);
        int64_t u = 0;
        if (nr <= 4)
            for (int64_t rt = 0; rt < nr; rt++) {
                int64_t lo, n;
                tile_keys(L, S, rt, lo, n);
                u += n;
            }
        for (uint32_t big = __ballot_sync(0xFFFFFFFFu, nr > 4); big; big &= big - 1) {
            const int l = __ffs(big) - 1;
            const seq_span X = { 0, __shfl_sync(0xFFFFFFFFu, S.n, l), __shfl_sync(0xFFFFFFFFu, S.kv, l) };
            const int64_t sum = units_by_warp(L, X);
            if (lane == l) u = sum;
        }
        mine += u;
    }
    if (tid < B_SUMS) C.sums[tid] = mine * P.n_head_kv;
    __syncthreads();
    int64_t W = 0;
    for (int i = lane; i < B_SUMS; i += 32) W += C.sums[i];
#pragma unroll
    for (int d = 16; d; d >>= 1) W += __shfl_xor_sync(0xFFFFFFFFu, W, d);
    const int64_t N = min((int64_t) gridDim.x, W);            // CTAs that get a share: one unit at least
    const bool work = blockIdx.x < N;
    if (work && warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" :: "r"(smem_addr(&C.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n");
    }
    tc_before();
    __syncthreads();
    tc_after();
    if (work) {
        const uint32_t tmem = C.tmem;
        uint32_t items = 0;                                   // handed out
        tile_item I;
        // the next item of warps 0 .. 9; false: the share is done, or the CTA gives up
        auto next_item = [&]() {
            const uint32_t i = items % B_ITEMS;
            if (!bar_wait_warp(it_full + 8 * i, (items / B_ITEMS) & 1, stop)) return false;
            I = C.item[i];
            __syncwarp();
            if (lane == 0) bar_arrive(it_empty + 8 * i);
            items++;
            return I.n > 0;
        };
        if (warp >= 8) {
            if constexpr (D == 128) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;\n" ::);
            if (warp == 10) {
                // ------------------------------------------------ items
                line_walk walk;
                walk.sums = C.sums;
                walk.per = per;
                walk.W = W;
                walk.N = N;
                walk.x = W * blockIdx.x / N;
                walk.x_end = W * (blockIdx.x + 1) / N;
                walk.base = walk.run_base = 0;
                walk.seq_len = -1;
                walk.run = walk.s = 0;
                do {
                    const uint32_t i = items % B_ITEMS;
                    walk.next(P, L, I);
                    if (!bar_wait_warp(it_empty + 8 * i, ((items / B_ITEMS) & 1) ^ 1, stop)) break;
                    if (lane == 0) {
                        C.item[i] = I;
                        bar_arrive(it_full + 8 * i);
                    }
                    __syncwarp();
                    items++;
                } while (I.n > 0);
            } else if (warp == 9) {
                // ------------------------------------------------ K and V pages
                const int box = min(1 << P.page_shift, B_KEYS), boxes = B_KEYS / box;
                uint32_t n = 0;                                  // buffers filled
                bool ok = true;
                while (ok && next_item()) {
                    const int seen = first_owned(I, L);
                    // the page (out of bounds: zeros) and its row that this lane copies of tile t
                    auto place = [&](int t, int & row) {
                        const int64_t key = (int64_t) I.key0 + t * B_KEYS + lane * box;
                        int64_t page = -1;
                        if (t < I.n && lane < boxes && key < I.kv && key + box > seen) page = page_of(P, I.seq, key);
                        row = (int) (key & ((1 << P.page_shift) - 1));
                        return (int) (page < 0 ? P.n_pages : page);
                    };
                    auto copy = [&](const CUtensorMap * map, int page, int row) {
                        const uint32_t b = n % ST;
                        if (!bar_wait_warp(kv_empty + 8 * b, ((n / ST) & 1) ^ 1, stop)) return false;
                        if (lane == 0) bar_expect(kv_full + 8 * b, TB);
                        __syncwarp();
                        if (lane < boxes)
#pragma unroll
                            for (int i = 0; i < HALVES; i++)
                                tma_page(ring + b * TB + i * HB + lane * box * 128, map, 64 * i, row, I.head, page, kv_full + 8 * b);
                        n++;
                        return true;
                    };
                    // in the order of their use: K 0 (K 1), then V 0, K 1 (K 2), V 1, ..
                    // (page ids are looked up a tile ahead)
                    int row[BUFS + 1], page[BUFS + 1];
#pragma unroll
                    for (int t = 0; t <= BUFS; t++) {
                        page[t] = place(t, row[t]);
                        if (t < BUFS && t < I.n) ok = ok && copy(&kmap, page[t], row[t]);
                    }
                    for (int t = 0; ok && t < I.n; t++) {
                        ok = copy(&vmap, page[0], row[0]);
                        if (t + BUFS < I.n) ok = ok && copy(&kmap, page[BUFS], row[BUFS]);
#pragma unroll
                        for (int i = 0; i < BUFS; i++) page[i] = page[i + 1], row[i] = row[i + 1];
                        page[BUFS] = place(t + BUFS + 1, row[BUFS]);
                    }
                }
                // nothing of this CTA's may be in flight when it ends
                give_up none = { 0, k_wait_cycles };
                for (uint32_t i = n > ST ? n - ST : 0; i < n; i++) (void) bar_wait(kv_full + 8 * (i % ST), (i / ST) & 1, &none);
            } else if (warp == 8) {
                // ------------------------------------------------ MMA
                uint32_t n = 0;                                  // ring position of the item's first K
                uint32_t tiles[2] = { 0, 0 }, nq[2] = { 0, 0 };  // tiles of each group so far; phases of q_full
                bool ok = true;
                while (ok && next_item()) {
                    const int groups = I.rows - I.r0 > B_ROWS ? 2 : 1;
                    const uint32_t nt = (uint32_t) I.n;
                    if (lane == 0) {
                        auto full = [&](uint32_t i) { return bar_wait(kv_full + 8 * (i % ST), (i / ST) & 1, stop); };
                        auto k_at = [&](uint32_t j) { return n + (j < BUFS ? j : 2 * j - BUFS + 1); };     // ring positions
                        auto v_at = [&](uint32_t j) { return n + min(j + BUFS, nt) + j; };
                        auto qk = [&](int g, uint32_t j) {
                            const uint32_t kb = ring + k_at(j) % ST * TB, qb = q_sm + g * QB, b = (tiles[g] + j) % BUFS;
#pragma unroll
                            for (int k = 0; k < D / 16; k++)
                                mma_ss(tmem + S_COL + 128 * g + 64 * b, smem_desc(qb + (k / 4) * QH + (k % 4) * 32, 16, 1024),
                                       smem_desc(kb + (k / 4) * HB + (k % 4) * 32, 16, 1024), idesc_qk, k > 0);
                            mma_commit(s_full + 16 * g + 8 * b);
                        };
                        for (uint32_t j = 0; ok && j < min(nt, (uint32_t) BUFS); j++) {
                            ok = full(k_at(j));
                            for (int g = 0; ok && g < groups; g++) {
                                if (j == 0) ok = bar_wait(q_full + 8 * g, nq[g]++ & 1, stop);
                                tc_after();
                                if (ok) qk(g, j);
                            }
                            if (ok) mma_commit(kv_empty + 8 * (k_at(j) % ST));
                        }
                        for (uint32_t j = 0; ok && j < nt; j++) {
                            const uint32_t vb = ring + v_at(j) % ST * TB;
                            ok = full(v_at(j));
                            for (int g = 0; ok && g < groups; g++) {
                                const uint32_t at = tiles[g] + j, b = at % BUFS;
                                auto pv = [&](int part) {
                                    if (!bar_wait(p_ready + 16 * g + 8 * (PARTS == 2 ? part : b), at / BUFS & 1, stop)) return false;
                                    tc_after();
#pragma unroll
                                    for (int kk = 4 * part; kk < 4 * part + 4; kk++)
                                        mma_ts(tmem + O_COL + D * g, tmem + S_COL + 128 * g + 64 * b + 8 * kk,
                                               smem_desc(vb + kk * 2048, HB, 1024), idesc_pv, j > 0 || kk > 0);
                                    return true;
                                };
                                if (!(ok = pv(0))) break;
                                if constexpr (PARTS == 2)
                                    if (!(ok = pv(1))) break;
                                if (j + 1 == nt) mma_commit(o_full + 8 * g);
                                else if (BUFS == 2) mma_commit(pv_done + 8 * g);
                                if (j + BUFS < nt) {
                                    if (g == 0 && !(ok = full(k_at(j + BUFS)))) break;
                                    qk(g, j + BUFS);
                                }
                            }
                            if (ok) {
                                mma_commit(kv_empty + 8 * (v_at(j) % ST));
                                if (j + BUFS < nt) mma_commit(kv_empty + 8 * (k_at(j + BUFS) % ST));
                            }
                        }
                        for (int g = 0; g < groups; g++) tiles[g] += nt;
                    }
                    n += 2 * nt;
                    ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
                }
                if (lane == 0) {
                    give_up none = { 0, k_wait_cycles };
                    mma_commit(drained);
                    (void) bar_wait(drained, 0, &none);
                }
                __syncwarp();
            }
        } else {
            if constexpr (D == 128) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;\n" ::);
            // ------------------------------------------------ softmax and output
            const int g = warp >> 2, row = tid & 127;
            const uint32_t lanes = (uint32_t) (warp & 3) << 21;      // TMEM lane 32 (warp % 4)
            const uint32_t s_at = tmem + lanes + S_COL + 128 * g, o_at = tmem + lanes + O_COL + D * g;
            uint32_t tiles = 0, no = 0, npv = 0;                     // tiles so far; phases of o_full and pv_done
            uint32_t n = 0;                                          // ring position of the item's first K
            const int win = (int) L.window;                          // below max_kv
            bool ok = true;
            for (; ok; items++) {
                // the item stays in shared memory: the loop over the keys needs its registers for the scores
                const uint32_t slot_i = items % B_ITEMS;
                if (!(ok = bar_wait_warp(it_full + 8 * slot_i, (items / B_ITEMS) & 1, stop))) break;
                const volatile tile_item & X = C.item[slot_i];
                const uint32_t nt = (uint32_t) X.n, ring0 = n;
                if (nt == 0) break;
                n += 2 * nt;
                auto release = [&] {
                    __syncwarp();
                    if (lane == 0) bar_arrive(it_empty + 8 * slot_i);
                };
                if (X.r0 + B_ROWS * g >= X.rows) {                   // no rows for this group
                    release();
                    continue;
                }
                auto my_row = [&] { return X.r0 + B_ROWS * g + row; };
                {
                    const int r = my_row();
                    const uint4 * src = reinterpret_cast<const uint4 *>(q + (int64_t) (X.first + r / L.G) * q_ld +
                                                                        (int64_t) (X.head * L.G + r % L.G) * D);
                    const uint32_t qb = q_sm + g * QB + row * 128;
                    const bool live = r < X.rows;
                    uint4 v[D / 8];
#pragma unroll
                    for (int i = 0; i < D / 8; i++) v[i] = live ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < D / 8; i++)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n"
                                     :: "r"(qb + (i / 8) * QH + (((i % 8) ^ (row & 7)) << 4)), "r"(v[i].x), "r"(v[i].y),
                                        "r"(v[i].z), "r"(v[i].w) : "memory");
                    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                    bar_arrive(q_full + 8 * g);
                }
                // a tile needs a look at its edges where its last key is past the first row's, or its first key before
                // the last row's window; rows of V that the sequence does not own lie only in such tiles
                const int first_pos = X.pos0 + (X.r0 + B_ROWS * g) / L.G - X.key0;
                const int last_win = win ? max(X.pos0 + (min(X.r0 + B_ROWS * g + B_ROWS, X.rows) - 1) / L.G, -1) - X.key0 - win : -1;
                float m = k_none, l = 0.0f;
                for (uint32_t j = 0; j < nt; j++) {
                    const uint32_t buf = tiles % BUFS, s_now = s_at + 64 * buf;
                    if (!(ok = bar_wait_warp(s_full + 16 * g + 8 * buf, tiles / BUFS & 1, stop))) break;
                    tiles++;
                    tc_after();
                    uint32_t sv[B_KEYS];
#pragma unroll
                    for (int i = 0; i < B_KEYS / 32; i++) tc_ld32(s_now + 32 * i, sv + 32 * i);
                    tc_wait_ld(sv);
                    if ((int) j * B_KEYS + B_KEYS - 1 > first_pos || (int) j * B_KEYS <= last_win) {
                        const int k0 = X.key0 + (int) j * B_KEYS, pos = X.pos0 + my_row() / L.G;
                        const int seen = win ? max(0, max(X.pos0, 0) - win + 1) : 0, kv = X.kv;
                        const int hi = pos - k0, lo = win ? pos - win + 1 - k0 : 0;     // columns lo .. hi
#pragma unroll
                        for (int i = 0; i < B_KEYS; i++)
                            if (i > hi || i < lo) sv[i] = 0xFF800000u;
                        // those rows of V may hold anything: weight 0 must meet 0
                        if (k0 + B_KEYS > kv || k0 < seen) {
                            const uint32_t i = ring0 + min(j + BUFS, nt) + j;
                            if (!(ok = bar_wait_warp(kv_full + 8 * (i % ST), (i / ST) & 1, stop))) break;
                            if (row < B_KEYS && (k0 + row >= kv || k0 + row < seen)) {
                                const uint32_t vb = ring + (i % ST) * TB + row * 128;
#pragma unroll
                                for (int c = 0; c < D / 8; c++)
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n"
                                                 :: "r"(vb + (c / 8) * HB + (c % 8) * 16), "r"(0) : "memory");
                            }
                            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
                        }
                    }
                    float t4[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
                    for (int i = 0; i < B_KEYS; i += 8)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            t4[e] = max3(t4[e], __uint_as_float(sv[i + 2 * e]), __uint_as_float(sv[i + 2 * e + 1]));
                    const float top = __fmul_rn(fmaxf(max3(t4[0], t4[1], t4[2]), t4[3]), scale_log2);     // rounded: never fused
                    if (__any_sync(0xFFFFFFFFu, top - m > lag)) {
                        const float mn = fmaxf(m, top - head), f = ex2(m - mn);
                        m = mn;
                        l *= f;
                        if (j > 0) {
                            // with two S, PV of the tile before may be on its way (with one, S came after it)
                            if (BUFS == 2 && !(ok = bar_wait_warp(pv_done + 8 * g, (npv - 1) & 1, stop))) break;
                            tc_after();
#pragma unroll
                            for (int i = 0; i < D / 32; i++) {
                                uint32_t ov[32];
                                tc_ld32(o_at + 32 * i, ov);
                                tc_wait_ld(ov);
#pragma unroll
                                for (int e = 0; e < 32; e++) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * f);
                                tc_st32(o_at + 32 * i, ov);
                            }
                        }
                    }
                    // past 2^22 the rounding of the reference's product, which the fused form puts into every exponent,
                    // passes 1/4: the scores' products are then rounded as well, and the largest is the reference again
                    float factor = scale_log2;
                    if (__any_sync(0xFFFFFFFFu, fabsf(m) > 0x1p22f && fabsf(m) < FLT_MAX)) {
                        if (fabsf(m) > 0x1p22f) {
                            factor = 1.0f;
#pragma unroll
                            for (int i = 0; i < B_KEYS; i++) sv[i] = __float_as_uint(__fmul_rn(__uint_as_float(sv[i]), scale_log2));
                        }
                        __syncwarp();
                    }
                    float2 add[2] = { { 0, 0 }, { 0, 0 } };
                    const float2 sc2 = make_float2(factor, factor), m2 = make_float2(-m, -m);
#pragma unroll
                    for (int i = 0; i < PARTS; i++) {
                        uint32_t pv[32];
#pragma unroll
                        for (int e = 0; e < 32; e++) {
                            const float2 x = fma2(make_float2(__uint_as_float(sv[64 * i + 2 * e]), __uint_as_float(sv[64 * i + 2 * e + 1])),
                                                  sc2, m2);
                            pv[e] = num<T>::pack(ex2(x.x), ex2(x.y));
                            add[e & 1] = add2(add[e & 1], num<T>::unpack(pv[e]));
                        }
                        tc_st32(s_now + 32 * i, pv);
                        tc_wait_st();
                        tc_before();
                        bar_arrive(p_ready + 16 * g + 8 * (PARTS == 2 ? i : buf));
                    }
                    npv += j + 1 < nt;         // PV of an item's last tile goes to o_full
                    l += (add[0].x + add[0].y) + (add[1].x + add[1].y);
                }
                if (!ok || !(ok = bar_wait_warp(o_full + 8 * g, no++ & 1, stop))) break;
                tc_after();
                const int r = my_row();
                const bool live = r < X.rows;
                const int64_t tok = X.first + r / L.G;
                const int head = X.head * L.G + r % L.G;
                // 32 dims at a time: o becomes the row's outputs
                auto put = [&](int i, uint32_t (&o)[32], float inv) {
                    uint4 * out = reinterpret_cast<uint4 *>(dst + tok * dst_ld + (int64_t) head * D + 32 * i);
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * inv);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        out[e] = make_uint4(pack2<T>(o[8 * e], o[8 * e + 1]), pack2<T>(o[8 * e + 2], o[8 * e + 3]),
                                            pack2<T>(o[8 * e + 4], o[8 * e + 5]), pack2<T>(o[8 * e + 6], o[8 * e + 7]));
                };
                const int c0 = X.c0, others = X.others;
                const bool cut_up = X.cut != 0;
                release();
                if (!cut_up) {
                    const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll 1
                    for (int i = 0; i < D / 32; i++) {
                        uint32_t o[32];
                        tc_ld32(o_at + 32 * i, o);
                        tc_wait_ld(o);
                        if (live) put(i, o, inv);
                    }
                    continue;
                }
                // [slot][warp 0..7][d / 4][lane] and [slot][warp][lane]
                auto slot = [&](int c) { return parts + ((int64_t) c * 2 + (c == c0)) * B_PART; };
                auto slot_o = [&](int c) { return reinterpret_cast<float4 *>(slot(c)) + warp * (D / 4) * 32 + lane; };
                auto slot_m = [&](int c) { return reinterpret_cast<float2 *>(slot(c) + B_TILE * 128) + warp * 32 + lane; };
#pragma unroll 1
                for (int i = 0; i < D / 32; i++) {
                    uint32_t o[32];
                    tc_ld32(o_at + 32 * i, o);
                    tc_wait_ld(o);
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        __stcg(slot_o(blockIdx.x) + (8 * i + e) * 32,
                               make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                                           __uint_as_float(o[4 * e + 3])));
                }
                __stcg(slot_m(blockIdx.x), make_float2(m, l));
                __threadfence();
                __syncwarp();
                int last = 0;
                if (lane == 0) last = atomicAdd(&counters[c0 * 8 + warp], 1) == others;
                if (!__shfl_sync(0xFFFFFFFFu, last, 0)) continue;
                __threadfence();
                m = k_none;
                l = 0.0f;
                for (int c = c0; c <= c0 + others; c++) {
                    const float2 ml = __ldcg(slot_m(c));
                    const float mn = fmaxf(m, ml.x);
                    l = l * ex2(m - mn) + ml.y * ex2(ml.x - mn);
                    m = mn;
                }
                const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll 1
                for (int i = 0; i < D / 32; i++) {
                    float a[32] = {};
                    for (int c = c0; c <= c0 + others; c++) {
                        const float f = ex2(__ldcg(slot_m(c)).x - m);
#pragma unroll
                        for (int e = 0; e < 8; e++) {
                            const float4 v = __ldcg(slot_o(c) + (8 * i + e) * 32);
                            a[4 * e] += v.x * f;
                            a[4 * e + 1] += v.y * f;
                            a[4 * e + 2] += v.z * f;
                            a[4 * e + 3] += v.w * f;
                        }
                    }
                    uint32_t o[32];
#pragma unroll
                    for (int e = 0; e < 32; e++) o[e] = __float_as_uint(a[e]);
                    if (live) put(i, o, inv);
                }
                if (lane == 0) counters[c0 * 8 + warp] = 0;
            }
            tc_wait_st();
        }
        __syncwarp();
    }
    tc_before();
    __syncthreads();
    if (work && warp == 8) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" :: "r"(C.tmem));
        if (lane == 0 && C.stop.stop) {
            atomicAdd(&g_paged_errors[1], 1ull);
            atomicAdd(ran_out, 1ull);
        }
    }
}

// ============================ sampling =====================================
//
// Where rows are fewer than SMs a cluster of CTAs takes a row and holds it in
// shared memory, each logit read once; where they are more, one CTA does and
// reads the row again in each step, from L2.  A warp has a contiguous part of
// the row, in order of index (CTA, warp, vector, lane, element).  What bounds it
// is instructions a logit where there are many rows, and the latencies of the
// steps and of the cluster's barriers where there are few.
//
// The sorted order is cut without sorting the row:
//   top-k    the k-th largest of the groups' maxima (a group: one place in one
//            thread's vectors) is a bound that the k largest logits pass; the
//            few that do go to a list, which is cut and finished;
//   min-p    the logits near enough to the maximum go to the list;
//   top-p    a histogram of the distance to the maximum bounds each bucket's
//            mass from its count, and so the cut's place to a few buckets; one
//            pass then takes the exact masses of all, of what lies above those
//            buckets, and the list of what lies in them;
//   a list that would be too long falls back to radix selection over the
//            32-bit order-preserving keys.
//
// Measured: 1 x 49,152 F32 with every filter 16 us, 48 rows of mixed filters 36
// us, 256 x 131,071 bf16 152 us (greedy rows alone 24, no filter 50, top-k 25-54,
// top-p alone 118-135: beside one pass of exponentials, as without a filter, it
// scans for the smallest logit and counts distances, one atomic a logit).
//
// Masses are integers of 2^-38 of the largest weight, rounded to nearest: sums
// are exact in any order, so the result hangs on no order of atomics.

constexpr int S_BUCKETS = 8192, S_COARSE = 1024, S_RADIX = 1024, S_LIST = 4096;
constexpr int k_row_ctas = 4;                   // of a cluster at most: a peer's memory is slow to read
constexpr float S_RANGE = 28.0f;               // exp(-28) < 2^-40: weightless
constexpr float S_UNIT = 0x1p-38f;

using ull = unsigned long long;

__device__ __forceinline__ uint32_t order_key(float x) {          // x is no NaN
    const uint32_t b = __float_as_uint(x + 0.0f);                 // -0 is 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}
// w in [0, 1] as hi 2^-15 + lo 2^-38: adding 1.5 2^8 leaves the multiple of
// 2^-15 in the low bits, adding 1.5 2^-15 to the remainder that of 2^-38
constexpr float S_HI = 384.0f, S_LO = 0x1.8p-15f;
__device__ __forceinline__ void mass_parts(float w, uint32_t & hi, uint32_t & lo) {
    const float h = w + S_HI, r = w - (h - S_HI);
    hi = __float_as_uint(h);
    lo = __float_as_uint(r + S_LO);
}
__device__ __forceinline__ ull mass_sum(uint32_t hi, uint32_t lo, int n) {  // of n parts added up
    const int h = (int) (hi - (uint32_t) n * 0x43C00000u), l = (int) (lo - (uint32_t) n * 0x38400000u);
    return (ull) (((long long) h << 23) + l);
}
__device__ __forceinline__ ull mass_of(float w) {
    uint32_t hi, lo;
    mass_parts(w, hi, lo);
    return mass_sum(hi, lo, 1);
}

__device__ __forceinline__ void mass_parts2(float2 w, uint32_t (&hi)[2], uint32_t (&lo)[2]) {
    const float2 h = add2(w, make_float2(S_HI, S_HI)), g = add2(h, make_float2(-S_HI, -S_HI));
    const float2 l = add2(add2(w, make_float2(-g.x, -g.y)), make_float2(S_LO, S_LO));
    hi[0] = __float_as_uint(h.x), hi[1] = __float_as_uint(h.y);
    lo[0] = __float_as_uint(l.x), lo[1] = __float_as_uint(l.y);
}

struct sample_row {
    float top, inv_t, top_p, min_p, u;
    int   k;
    bool  greedy;
    __device__ void read(int64_t row, int V, const float * temperature, const int32_t * top_k, const float * p, const float * m,
                         const float * uniform) {
        const float t = temperature ? temperature[row] : 1.0f;
        greedy = !(t > 0.0f);
        inv_t = fminf(1.0f / t, FLT_MAX);
        k = top_k ? top_k[row] : 0;
        if (k <= 0 || k > V) k = V;
        top_p = p ? p[row] : 1.0f;
        min_p = m ? fminf(m[row], 1.0f) : 0.0f;                   // the largest always stays
        if (min_p != min_p) min_p = 0.0f;
        u = uniform[row];
    }
    // NaN and what is too far below: no weight
    __device__ __forceinline__ float weight(float v) const { return expf(fmaxf((v - top) * inv_t, -100.0f)); }
    __device__ __forceinline__ float2 distance2(float a, float b) const {
        return add2(make_float2(a, b), make_float2(-top, -top));
    }
    __device__ __forceinline__ float2 weight2(float2 d) const {
        const float2 z = mul2(d, make_float2(inv_t, inv_t));
        return make_float2(expf(fmaxf(z.x, -100.0f)), expf(fmaxf(z.y, -100.0f)));
    }
    __device__ __forceinline__ ull mass(float v) const { return mass_of(weight(v)); }
    // the masses' limit: what lies before a kept token stays at or below it
    __device__ ull mass_limit(ull whole) const {
        const double want = ceil((double) top_p * (double) whole);
        return want >= 1.0 ? (ull) want - 1 : 0ull;
    }
    __device__ ull goal(ull total) const {
        const ull g = (ull) ((double) fminf(fmaxf(u, 0.0f), 1.0f) * (double) total);
        return g < total ? g : total - 1;
    }
    __device__ float prob(float w, ull total) const { return (float) ((double) w / ((double) total * (double) S_UNIT)); }
};

struct alignas(16) sample_smem {   // the row's vectors follow it
    ull      list[S_LIST];           // key << 32 | ~index: the sorted order
    uint32_t hist[S_BUCKETS];      // counts, or four 11-bit parts of the masses of S_RADIX buckets
    ull      scan[33], ends[32], part_mass[32];
    uint32_t part_ties[32];
    uint32_t list_mass[3][k_row_ctas * 32], list_ties[k_row_ctas * 32];   // CTA 0: what the list adds to the parts
    ull      shared[2][2];         // sums that the cluster adds up, two uses in turn
    float    hi[32], lo[32], top, low;
    uint32_t key_lo, key_hi;
    int      n, best, first, b1, b2, at;
    ull      above, goal, ties, total, v_lo, v_hi;
    float    cut;
};

// inclusive scan over the block, total in total
template <int WARPS, class V>
__device__ __forceinline__ V block_scan(V v, V * sums, V & total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const V o = __shfl_up_sync(0xFFFFFFFFu, v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    V s = lane < WARPS ? sums[lane] : V(0), run = s;
#pragma unroll
    for (int d = 1; d < WARPS; d <<= 1) {
        const V o = __shfl_up_sync(0xFFFFFFFFu, run, d);
        if (lane >= d) run += o;
    }
    total = __shfl_sync(0xFFFFFFFFu, run, WARPS - 1);
    return v + __shfl_sync(0xFFFFFFFFu, run - s, warp);
}
template <int WARPS, class V>
__device__ __forceinline__ V block_sum(V v, V * sums) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
    __syncthreads();
    V t = 0;
#pragma unroll
    for (int w = 0; w < WARPS; w++) t += sums[w];
    return t;
}
// Of the block's items (those with m > 0, all v different) in falling order of
// v: the last one that has at most `limit` of m before it.  A histogram over
// the items' range, 1024-fold finer each time, until one item is left.
template <int THREADS, int PER, class S>
__device__ __forceinline__ ull block_select(const ull (&v)[PER], const ull (&m)[PER], ull limit, S & M) {
    constexpr int PR = S_RADIX / THREADS;
    const int tid = threadIdx.x, lane = tid & 31;
    ull lo = ~0ull, hi = 0, above = 0;
#pragma unroll
    for (int j = 0; j < PER; j++)
        if (m[j]) {
            lo = min(lo, v[j]);
            hi = max(hi, v[j]);
        }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d));
        hi = max(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
    }
    __syncthreads();
    if (lane == 0) {
        M.scan[tid >> 5] = lo;
        M.ends[tid >> 5] = hi;
    }
    __syncthreads();
    lo = lane < THREADS / 32 ? M.scan[lane] : ~0ull;
    hi = lane < THREADS / 32 ? M.ends[lane] : 0ull;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        lo = min(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, d));
        hi = max(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, d));
    }
    while (lo < hi) {
        const ull span = hi - lo;
        const int shift = span < S_RADIX ? 0 : 54 - __clzll(span);
        for (int i = tid; i < 2 * S_RADIX; i += THREADS) M.hist[i] = 0;
        if (tid == 0) {
            M.best = -1;
            M.v_lo = ~0ull;
            M.v_hi = 0;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (m[j] && v[j] >= lo && v[j] <= hi) {               // 4096 items of 2^38: two sums of 19 bits each
                const int b = (int) ((hi - v[j]) >> shift);
                atomicAdd(&M.hist[b], (uint32_t) m[j] & 0x7FFFFu);
                if (m[j] >> 19) atomicAdd(&M.hist[S_RADIX + b], (uint32_t) (m[j] >> 19));
            }
        __syncthreads();
        ull c[PR], sum = 0, t;
#pragma unroll
        for (int j = 0; j < PR; j++) {
            c[j] = M.hist[PR * tid + j] + ((ull) M.hist[S_RADIX + PR * tid + j] << 19);
            sum += c[j];
        }
        ull run = above + block_scan<THREADS / 32>(sum, M.scan, t) - sum, at[PR];
        int best = -1;
#pragma unroll
        for (int j = 0; j < PR; j++) {
            at[j] = run;
            if (c[j] && run <= limit) best = PR * tid + j;
            run += c[j];
        }
        best = __reduce_max_sync(0xFFFFFFFFu, best);
        if (lane == 0 && best >= 0) atomicMax(&M.best, best);
        __syncthreads();
        best = M.best;
#pragma unroll
        for (int j = 0; j < PR; j++)
            if (PR * tid + j == best) M.above = at[j];
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (m[j] && v[j] >= lo && v[j] <= hi && (int) ((hi - v[j]) >> shift) == best) {
                atomicMin(&M.v_lo, v[j]);
                atomicMax(&M.v_hi, v[j]);
            }
        __syncthreads();
        lo = M.v_lo;
        hi = M.v_hi;
        above = M.above;
        __syncthreads();
    }
    return hi;
}

// falling order over the threads below `size` (a power of two from 32 on); the
// other warps take no part
__device__ __forceinline__ ull block_sort(ull v, int size, ull * a) {
    const int tid = threadIdx.x;
    if (tid >= size) return v;
    auto sync = [&] { asm volatile("bar.sync 1, %0;\n" :: "r"(size) : "memory"); };
    for (int run = 2; run <= size; run <<= 1)
        for (int d = run >> 1; d; d >>= 1) {
            ull o;
            if (d < 32) {
                o = __shfl_xor_sync(0xFFFFFFFFu, v, d);
            } else {
                sync();
                a[tid] = v;
                sync();
                o = a[tid ^ d];
            }
            const bool larger = ((tid & run) == 0) == ((tid & d) == 0);
            v = larger ? max(v, o) : min(v, o);
        }
    return v;
}

template <class T> struct vec16;
template <> struct vec16<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ float at(const uint4 & v, int e) {
        return __uint_as_float(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w);
    }
    static __device__ __forceinline__ float top(const uint4 & r) { return fmaxf(fmaxf(at(r, 0), at(r, 1)), fmaxf(at(r, 2), at(r, 3))); }
    // the maximum of each place in the vectors; NaN counts for nothing
    template <class Each> static __device__ __forceinline__ void maxima(Each each, float (&top)[N]) {
#pragma unroll
        for (int e = 0; e < N; e++) top[e] = -INFINITY;
        each([&](const uint4 & r, int) {
#pragma unroll
            for (int e = 0; e < N; e++) top[e] = fmaxf(top[e], at(r, e));
        });
    }
};
template <class T> struct vec16 {
    static constexpr int N = 8;
    static __device__ __forceinline__ float at(const uint4 & v, int e) {
        const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(e & 1 ? w & 0xFFFF0000u : w << 16);
        const uint16_t h = (uint16_t) (e & 1 ? w >> 16 : w & 0xFFFF);
        return num<T>::to(*reinterpret_cast<const T *>(&h));
    }
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    static __device__ __forceinline__ float top(const uint4 & r) {
        const T2 a = __hmax2(__hmax2(*reinterpret_cast<const T2 *>(&r.x), *reinterpret_cast<const T2 *>(&r.y)),
                             __hmax2(*reinterpret_cast<const T2 *>(&r.z), *reinterpret_cast<const T2 *>(&r.w)));
        return num<T>::to(__hmax(a.x, a.y));
    }
    template <class Each> static __device__ __forceinline__ void maxima(Each each, float (&top)[N]) {
        const T none = num<T>::from(-INFINITY);
        T2 m[4];
#pragma unroll
        for (int e = 0; e < 4; e++) m[e] = T2(none, none);
        each([&](const uint4 & r, int) {
            const uint32_t w[4] = { r.x, r.y, r.z, r.w };
#pragma unroll
            for (int e = 0; e < 4; e++) m[e] = __hmax2(m[e], *reinterpret_cast<const T2 *>(&w[e]));
        });
#pragma unroll
        for (int e = 0; e < 4; e++) {
            top[2 * e] = num<T>::to(m[e].x);
            top[2 * e + 1] = num<T>::to(m[e].y);
        }
    }
};

template <class T, int THREADS, bool HELD>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
k_sample(const T * __restrict__ logits, int64_t ld, int V, int vecs, int C, const float * __restrict__ temperature,
         const int32_t * __restrict__ top_k, const float * __restrict__ top_p, const float * __restrict__ min_p,
         const float * __restrict__ u, int32_t * __restrict__ token, float * __restrict__ prob) {
    constexpr int E = vec16<T>::N, WARPS = THREADS / 32, PER = S_LIST / THREADS;
    extern __shared__ __align__(16) unsigned char sample_sm[];
    using smem = sample_smem;
    smem & M = *reinterpret_cast<smem *>(sample_sm);
    const int64_t row = blockIdx.x / C;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int cta = HELD ? (int) (blockIdx.x % C) : 0;            // the cluster is the row's C CTAs in order
    auto peer = [&](int c) -> smem & {
        if constexpr (HELD) return *cg::this_cluster().map_shared_rank(&M, c);
        return M;
    };
    auto csync = [&] {
        if (HELD && C > 1) cg::this_cluster().sync();
        else __syncthreads();
    };
    const T * x = logits + row * ld;
    const int lead = (int) (reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));    // vectors start at 16-byte boundaries
    // vector i of the row, 32 lanes of E elements: warp w of CTA c has vecs of them from (c * WARPS + w) * vecs on
    const int origin = lane * E - lead, w_first = (cta * WARPS + warp) * vecs;
    uint4 * const held = reinterpret_cast<uint4 *>(sample_sm + sizeof(smem)) + lane;
    auto ends = [&](int at) {                  // a vector at the row's ends: -inf beyond them
        alignas(16) T t[E];
#pragma unroll
        for (int e = 0; e < E; e++) t[e] = at + e >= 0 && at + e < V ? x[at + e] : num<T>::from(-INFINITY);
        return *reinterpret_cast<const uint4 *>(t);
    };
    auto fetch = [&](int i) {
        if constexpr (HELD) return held[(i - cta * WARPS * vecs) * 32];
        const int at = origin + i * 32 * E;
        if (at >= 0 && at + E <= V) return __ldg(reinterpret_cast<const uint4 *>(x + at));
        return ends(at);
    };
    // f(vector, index of its first element) for the row's vectors from .. to - 1; from memory two at a
    // time (eight copies of f spent a third of the time on fetching instructions: 218 against 151 us on 256 x 131,071)
    auto each_vec = [&](int from, int to, auto f) {
        constexpr int N = HELD ? 1 : 2;
        for (int i = from; i < to; i += N) {
            uint4 r[N];
#pragma unroll
            for (int j = 0; j < N; j++)
                if (i + j < to) r[j] = fetch(i + j);
#pragma unroll
            for (int j = 0; j < N; j++)
                if (i + j < to) f(r[j], origin + (i + j) * 32 * E);
        }
    };
    // f(value, index, its place in the vector) for this warp's part
    auto each = [&](auto f) {
        each_vec(w_first, w_first + vecs, [&](const uint4 & r, int at) {
#pragma unroll
            for (int e = 0; e < E; e++) f(vec16<T>::at(r, e), at + e, e);
        });
    };
    // sums over the cluster's threads
    int turn = 0;
    auto cluster_sum = [&](ull a, ull b, ull & all_a, ull & all_b) {
        a = block_sum<WARPS>(a, M.scan);
        b = block_sum<WARPS>(b, M.scan);
        if (tid == 0) {
            M.shared[turn][0] = a;
            M.shared[turn][1] = b;
        }
        csync();
        all_a = lane < C ? peer(lane).shared[turn][0] : 0ull;     // side by side: a peer's memory is far
        all_b = lane < C ? peer(lane).shared[turn][1] : 0ull;
#pragma unroll
        for (int d = 1; d < k_row_ctas; d <<= 1) {
            all_a += __shfl_xor_sync(0xFFFFFFFFu, all_a, d);
            all_b += __shfl_xor_sync(0xFFFFFFFFu, all_b, d);
        }
        all_a = __shfl_sync(0xFFFFFFFFu, all_a, 0);
        all_b = __shfl_sync(0xFFFFFFFFu, all_b, 0);
        turn ^= 1;
    };
    pdl_entry();
    if constexpr (HELD) {
        for (int i = 0; i < vecs; i++) {
            const int at = origin + (w_first + i) * 32 * E;
            uint4 * to = held + (warp * vecs + i) * 32;
            if (at >= 0 && at + E <= V) cp16(smem_addr(to), x + at, true);
            else *to = ends(at);
        }
        cp_commit();
    }
    sample_row R;
    R.read(row, V, temperature, top_k, top_p, min_p, u);
    for (int i = tid; i < S_BUCKETS; i += THREADS) M.hist[i] = 0;
    for (int i = tid; i < 3 * k_row_ctas * 32; i += THREADS) (&M.list_mass[0][0])[i] = 0;
    for (int i = tid; i < k_row_ctas * 32; i += THREADS) M.list_ties[i] = 0;
    if (tid == 0) {
        M.n = 0;
        M.first = 0x7FFFFFFF;
        M.b1 = M.b2 = S_BUCKETS;
        M.key_lo = 0xFFFFFFFFu;
        M.key_hi = 0;
    }
    if constexpr (HELD) cp_wait<0>();          // a lane reads only what it has fetched, until the barrier

    // ---- the largest and the smallest finite logit, and the groups' maxima
    float group[E], low = INFINITY, top = -INFINITY;
    vec16<T>::maxima([&](auto f) { each_vec(w_first, w_first + vecs, f); }, group);
#pragma unroll
    for (int g = 0; g < E; g++) top = fmaxf(top, group[g]);
    if (R.top_p < 1.0f && !R.greedy) each([&](float v, int, int) { low = fminf(low, v == -INFINITY ? INFINITY : v); });
    auto warp_ends = [&] {
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
            low = fminf(low, __shfl_xor_sync(0xFFFFFFFFu, low, d));
        }
    };
    warp_ends();
    if (lane == 0) {
        M.hi[warp] = top;
        M.lo[warp] = low;
    }
    __syncthreads();
    top = lane < WARPS ? M.hi[lane] : -INFINITY;
    low = lane < WARPS ? M.lo[lane] : INFINITY;
    warp_ends();
    if (HELD && C > 1) {
        if (tid == 0) {
            M.top = top;
            M.low = low;
        }
        csync();
        if (lane < C) {
            top = peer(lane).top;
            low = peer(lane).low;
        }
        warp_ends();
    }
    R.top = top + 0.0f;
    if (top == -INFINITY || R.greedy) {
        int at = 0x7FFFFFFF;
        if (top != -INFINITY) each([&](float v, int i, int) {
            if (v == top) at = min(at, i);
        });
        at = __reduce_min_sync(0xFFFFFFFFu, at);
        if (lane == 0 && at != 0x7FFFFFFF) atomicMin(&peer(0).first, at);
        csync();
        if (cta == 0 && tid == 0) {
            token[row] = top == -INFINITY ? -1 : M.first;
            if (prob) prob[row] = top == -INFINITY ? 0.0f : 1.0f;
        }
        return;
    }

    // kept: above `cut`, and the first `ties` equal to it
    float cut = -INFINITY;
    ull ties = 0, whole = 0;
    const bool by_k = R.k < V, by_p = R.top_p < 1.0f;

    // ---- CTA 0: the list, cut and finished.  `above`: the mass before it, whose tokens stay; with `open` the tokens
    // above the list are not in it: the cut is found, and what is kept is left to the steps below
    auto set_cut = [&](uint32_t key, int kept_equal) {
        cut = key_value(key);
        for (int i = tid; i < k_row_ctas * 32; i += THREADS) M.list_mass[0][i] = M.list_mass[1][i] = M.list_mass[2][i] = M.list_ties[i] = 0;
        ties = block_sum<WARPS>(kept_equal, reinterpret_cast<int *>(M.scan));
    };
    // a kept token of the list counts for its warp; 4096 masses in three 14-bit parts fit 32 bits
    auto add_to_part = [&](ull token_key, float w) {
        const int part = (int) (~(uint32_t) token_key + lead) / (vecs * 32 * E);
        if (key_value((uint32_t) (token_key >> 32)) == cut) {
            atomicAdd(&M.list_ties[part], 1u);
        } else {
            const ull m = mass_of(w);
            atomicAdd(&M.list_mass[0][part], (uint32_t) m & 0x3FFFu);
            if (m >> 14) atomicAdd(&M.list_mass[1][part], (uint32_t) (m >> 14) & 0x3FFFu);
            if (m >> 28) atomicAdd(&M.list_mass[2][part], (uint32_t) (m >> 28));
        }
    };
    auto finish_sorted = [&](int n, ull above, bool open) {       // n <= THREADS: one token a thread
        int size = 32;
        while (size < n) size <<= 1;
        const ull mine = tid < n ? M.list[tid] : 0ull;
        __syncthreads();                       // the list's place is free
        ull a = block_sort(mine, size, M.list), total;
        float w = a ? R.weight(key_value((uint32_t) (a >> 32))) : 0.0f;
        ull m = a && tid < R.k ? mass_of(w) : 0ull;
        const ull run = above + block_scan<WARPS>(m, M.scan, total) - m;
        if (by_k) whole = total;
        const bool keep = a && tid < R.k && (!by_p || run <= R.mass_limit(whole)) && w >= R.min_p;
        if (open) {
            const int all = __syncthreads_count(keep);            // the list's first ones
            if (all == 0) return;                                 // min_p: nothing of the list stays
            if (tid == all - 1) M.key_lo = (uint32_t) (a >> 32);
            __syncthreads();
            const uint32_t key = M.key_lo;
            set_cut(key, keep && (uint32_t) (a >> 32) == key);
            if (keep) add_to_part(a, w);
            return;
        }
        // ~index first: falling in order of index
        a = block_sort(keep ? (ull) (uint32_t) a << 32 | (uint32_t) (a >> 32) : 0ull, size, M.list);
        w = a ? R.weight(key_value((uint32_t) a)) : 0.0f;
        m = a ? mass_of(w) : 0ull;
        const ull upto = block_scan<WARPS>(m, M.scan, total), goal = R.goal(total);
        if (m && goal < upto && goal >= upto - m) {
            token[row] = (int32_t) ~(uint32_t) (a >> 32);
            if (prob) prob[row] = R.prob(w, total);
        }
    };
    auto finish_selected = [&](int n, ull above, bool open) {
        ull a[PER], m[PER];
        float w[PER];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int i = tid + j * THREADS;
            a[j] = i < n ? M.list[i] : 0ull;
            w[j] = i < n ? R.weight(key_value((uint32_t) (a[j] >> 32))) : 0.0f;
            m[j] = i < n ? 1ull : 0ull;
        }
        auto cut_off = [&](ull limit) {
            const ull last = block_select<THREADS>(a, m, limit, M);
#pragma unroll
            for (int j = 0; j < PER; j++)
                if (a[j] < last) a[j] = 0;
        };
        if (by_k && n > R.k) cut_off((ull) R.k - 1);
        ull sum = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) sum += m[j] = a[j] ? mass_of(w[j]) : 0ull;
        if (by_k) whole = block_sum<WARPS>(sum, M.scan);
        if (by_p) cut_off(max(R.mass_limit(whole), above) - above);
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (!(w[j] >= R.min_p)) a[j] = 0;
        if (open) {
            uint32_t key = 0xFFFFFFFFu;
#pragma unroll
            for (int j = 0; j < PER; j++)
                if (a[j]) key = min(key, (uint32_t) (a[j] >> 32));
            key = __reduce_min_sync(0xFFFFFFFFu, key);
            __syncthreads();
            if (tid == 0) M.key_lo = 0xFFFFFFFFu;
            __syncthreads();
            if (lane == 0) atomicMin(&M.key_lo, key);
            __syncthreads();
            key = M.key_lo;
            if (key == 0xFFFFFFFFu) return;
            int eq = 0;
#pragma unroll
            for (int j = 0; j < PER; j++) eq += a[j] && (uint32_t) (a[j] >> 32) == key;
            set_cut(key, eq);
#pragma unroll
            for (int j = 0; j < PER; j++)
                if (a[j]) add_to_part(a[j], w[j]);
            return;
        }
        sum = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            sum += m[j] = a[j] ? mass_of(w[j]) : 0ull;
            a[j] = (uint32_t) a[j];
        }
        const ull total = block_sum<WARPS>(sum, M.scan);
        const ull pick = block_select<THREADS>(a, m, R.goal(total), M);
#pragma unroll
        for (int j = 0; j < PER; j++)
            if (m[j] && a[j] == pick) {
                token[row] = (int32_t) ~(uint32_t) pick;
                if (prob) prob[row] = R.prob(w[j], total);
            }
    };
    // the list (n tokens, with `apart` in the CTAs' own lists), finished by CTA 0; true: the row is done
    auto finish = [&](int n, ull above, bool open, bool apart) {
        if (apart && cta == 0 && C > 1) {
            // warp w copies of CTA w % C
            const int nc = lane < C ? peer(lane).n : 0, c = warp % C;
            int at = 0;
            for (int r = 0; r < c; r++) at += __shfl_sync(0xFFFFFFFFu, nc, r);
            const int mine = __shfl_sync(0xFFFFFFFFu, nc, c);
            if (c > 0)
                for (int i = warp / C * 32 + lane; i < mine; i += WARPS / C * 32) M.list[at + i] = peer(c).list[i];
        }
        if (apart) csync();                    // CTA 0 has them all
        if (cta == 0) {
            if (n <= THREADS) finish_sorted(n, above, open);
            else finish_selected(n, above, open);
            if (open && tid == 0) {
                M.cut = cut;
                M.ties = ties;
            }
        }
        if (!open) {
            if (HELD && C > 1 && cta == 0) cg::this_cluster().sync();    // the others have read its memory, and are gone
            return true;
        }
        csync();
        cut = peer(0).cut;
        ties = peer(0).ties;
        return false;
    };
    auto push = [&](float v, int i) {
        const int at = atomicAdd(&M.n, 1);
        if (at < S_LIST) M.list[at] = (ull) order_key(v) << 32 | (uint32_t) ~i;
    };
    auto listed = [&] {                        // after a barrier
        return (int) __reduce_add_sync(0xFFFFFFFFu, lane < C ? (uint32_t) min(peer(lane).n, S_LIST + 1) : 0u);
    };

    bool found = false;                        // cut and ties are known
    bool parts_known = false;                  // and the warps' masses: above the list in part_mass, the list's in list_mass
    if (top == INFINITY || (by_p && low >= top)) {
        // nothing but the maximum has a weight, or every logit is the maximum
        ull eq = 0, none;
        each([&](float v, int, int) { eq += v == top; });
        cluster_sum(eq, 0, eq, none);
        ties = min(eq, (ull) R.k);
        if (by_p) ties = max(1ull, min(ties, (ull) ceil((double) R.top_p * (double) ties)));
        cut = top;
        found = true;
    } else if (by_k || by_p || R.min_p > 0.0f) {
        // distance to the maximum in buckets: up to the smallest logit, or to where nothing weighs
        const float reach = fminf(low < top ? top - low : INFINITY, S_RANGE / R.inv_t);
        // finite, so that the maximum's own place is 0: below a reach of 2.4e-35 the logits take fewer buckets
        const float q = -fminf((S_BUCKETS - 1) / reach, FLT_MAX);
        auto place = [&](float v) { return (v - top) * q; };      // NaN, or S_BUCKETS and more: none
        float below = 0.0f;                                       // the list: place < below
        bool list = false;
        if (by_k) {
            // every group's maximum is a logit: where k of them are, k logits are
#pragma unroll
            for (int g = 0; g < E; g++) {
                const float b = place(group[g]);
                if (b < S_BUCKETS) atomicAdd(&M.hist[(int) b / (S_BUCKETS / S_COARSE)], 1u);
            }
            csync();
            // every CTA adds up the cluster's histograms for itself
            constexpr int PB = (S_COARSE + THREADS - 1) / THREADS;
            uint32_t c[PB] = {}, sum = 0, all, h[PB][k_row_ctas];
#pragma unroll
            for (int j = 0; j < PB; j++)
#pragma unroll
                for (int r = 0; r < k_row_ctas; r++)
                    if (r < C) h[j][r] = peer(r).hist[PB * tid + j];
#pragma unroll
            for (int j = 0; j < PB; j++) {
#pragma unroll
                for (int r = 0; r < k_row_ctas; r++)
                    if (r < C) c[j] += h[j][r];
                sum += c[j];
            }
            uint32_t run = block_scan<WARPS>(sum, reinterpret_cast<uint32_t *>(M.scan), all) - sum;
            int b1 = S_COARSE;
#pragma unroll
            for (int j = 0; j < PB; j++) {
                run += c[j];
                if (run >= (uint32_t) R.k) b1 = min(b1, PB * tid + j);
            }
            b1 = __reduce_min_sync(0xFFFFFFFFu, b1);
            if (lane == 0) atomicMin(&M.b1, b1);
            __syncthreads();
            below = (float) min(S_BUCKETS, (M.b1 + 1) * (S_BUCKETS / S_COARSE));
            list = true;
        } else if (by_p) {
            // a CTA that holds its part has less than 2^16 logits: two counts to a word, for the cluster's sake
            each([&](float v, int, int) {
                const float b = place(v);
                if (b < S_BUCKETS) {
                    if (HELD) atomicAdd(&M.hist[(int) b >> 1], (int) b & 1 ? 0x10000u : 1u);
                    else atomicAdd(&M.hist[(int) b], 1u);
                }
            });
        } else {
            // exp(-d) >= min_p, with room for exp's and the logarithm's rounding
            below = fminf((float) S_BUCKETS, (1e-3f - logf(R.min_p)) / R.inv_t * -q + 1.0f);
            list = true;
        }
        if (!list) {
            csync();
            constexpr int PB = S_BUCKETS / THREADS;
            uint32_t c[PB] = {};
            if constexpr (HELD) {
                uint4 h[PB / 8][k_row_ctas];
#pragma unroll
                for (int j = 0; j < PB / 8; j++)
#pragma unroll
                    for (int r = 0; r < k_row_ctas; r++)
                        if (r < C) h[j][r] = reinterpret_cast<const uint4 *>(peer(r).hist + PB / 2 * tid)[j];
#pragma unroll
                for (int j = 0; j < PB / 8; j++)
#pragma unroll
                    for (int r = 0; r < k_row_ctas; r++)
                        if (r < C) {
                            const uint32_t w[4] = { h[j][r].x, h[j][r].y, h[j][r].z, h[j][r].w };
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                c[8 * j + 2 * e] += w[e] & 0xFFFFu;
                                c[8 * j + 2 * e + 1] += w[e] >> 16;
                            }
                        }
            } else {
#pragma unroll
                for (int j = 0; j < PB; j++) c[j] = M.hist[PB * tid + j];
            }
            // each bucket's mass lies between count x its ends' weights; 1e-4 for the rounding of places and sums
            const float step = R.inv_t / -q, ratio = expf(-step), w_first_bucket = expf(-step * (PB * tid));
            float least = 0, most = 0, all_least, all_most, wb = w_first_bucket;
#pragma unroll
            for (int j = 0; j < PB; j++) {
                most += c[j] * wb;
                wb *= ratio;
                least += c[j] * wb;
            }
            float * fs = reinterpret_cast<float *>(M.scan);
            const float least_upto = block_scan<WARPS>(least, fs, all_least);
            float lower = least_upto - least, upper = block_scan<WARPS>(most, fs, all_most) - most;
            int b1 = S_BUCKETS, b2 = S_BUCKETS;
            wb = w_first_bucket;
#pragma unroll
            for (int j = 0; j < PB; j++) {
                upper += c[j] * wb;
                wb *= ratio;
                lower += c[j] * wb;
                if (upper * 1.0001f >= R.top_p * all_least * 0.9999f) b1 = min(b1, PB * tid + j);
                if (lower * 0.9999f >= R.top_p * all_most * 1.0001f) b2 = min(b2, PB * tid + j);
            }
            b1 = __reduce_min_sync(0xFFFFFFFFu, b1);
            b2 = __reduce_min_sync(0xFFFFFFFFu, b2);
            if (lane == 0) {
                atomicMin(&M.b1, b1);
                atomicMin(&M.b2, b2);
            }
            __syncthreads();
            b1 = M.b1 == S_BUCKETS ? 0 : M.b1;
            b2 = min(M.b2, S_BUCKETS - 1);
            // all down to the cut's buckets, if they are few, else the cut's buckets
            uint32_t upto = 0;
#pragma unroll
            for (int j = 0; j < PB; j++) upto += PB * tid + j <= b2 ? c[j] : 0u;
            upto = block_sum<WARPS>(upto, reinterpret_cast<uint32_t *>(M.scan));
            const float from = upto <= S_LIST ? 0.0f : (float) b1, to = (float) b2 + 1.0f;
            ull all_m = 0, above_m = 0, above;
            uint32_t klo = 0xFFFFFFFFu, khi = 0;
            each_vec(w_first, w_first + vecs, [&](const uint4 & r, int at) {
                uint32_t hi = 0, lo = 0, ahi = 0, alo = 0;
                int an = 0;
                bool some = false;
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float2 d = R.distance2(vec16<T>::at(r, e), vec16<T>::at(r, e + 1)), b2 = mul2(d, make_float2(q, q));
                    uint32_t h[2], l[2];
                    mass_parts2(R.weight2(d), h, l);
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float b = j ? b2.y : b2.x;
                        const bool over = b < from;
                        hi += h[j];
                        lo += l[j];
                        ahi += over ? h[j] : 0u;
                        alo += over ? l[j] : 0u;
                        an += over;
                        some |= !over && b < to;
                    }
                }
                all_m += mass_sum(hi, lo, E);
                above_m += mass_sum(ahi, alo, an);
                if (some) {
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const float v = vec16<T>::at(r, e), b = place(v);
                        if (b >= from && b < to) {
                            klo = min(klo, order_key(v));
                            khi = max(khi, order_key(v));
                            if (*(volatile int *) &M.n <= S_LIST) push(v, at + e);
                        }
                    }
                }
            });
            klo = __reduce_min_sync(0xFFFFFFFFu, klo);
            khi = __reduce_max_sync(0xFFFFFFFFu, khi);
            if (lane == 0) {
                atomicMin(&M.key_lo, klo);
                atomicMax(&M.key_hi, khi);
            }
            {
                ull m = above_m;
#pragma unroll
                for (int d = 16; d; d >>= 1) m += __shfl_xor_sync(0xFFFFFFFFu, m, d);
                if (lane == 0) M.part_mass[warp] = m;
            }
            cluster_sum(all_m, above_m, whole, above);
            const int n = listed();
            if (n <= S_LIST) {
                if (finish(n, above, from > 0.0f, true)) return;
                found = true;
                parts_known = R.min_p <= 0.0f;
            }
            if (tid == 0) M.above = above;
        }
        if (list) {
            smem & M0 = peer(0);               // into CTA 0's list
            bool room = true;
            each_vec(w_first, w_first + vecs, [&](const uint4 & r, int at) {
                if (place(vec16<T>::top(r)) < below && room) {    // rarely
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const float v = vec16<T>::at(r, e);
                        if (place(v) < below && room) {
                            const int i = atomicAdd(&M0.n, 1);
                            if (i < S_LIST) M0.list[i] = (ull) order_key(v) << 32 | (uint32_t) ~(at + e);
                            else room = false;
                        }
                    }
                }
            });
            csync();
            const int n = M0.n;
            if (n <= S_LIST) {
                finish(n, 0, false, false);
                return;
            }
        }
        // ---- radix selection, by count for top-k, by mass for top-p
        for (int by_mass = 0; by_mass < 2 && !found; by_mass++) {
            if (by_mass ? !by_p : !by_k) continue;
            const bool after_k = by_mass && by_k;
            uint32_t key_lo = 0x00800000u, key_hi = order_key(top);   // above -inf
            ull above = 0, limit = (ull) (R.k - 1);
            csync();
            if (by_mass && !by_k) {
                for (int c = 0; c < C; c++) {
                    key_lo = c ? min(key_lo, peer(c).key_lo) : peer(c).key_lo;
                    key_hi = c ? max(key_hi, peer(c).key_hi) : peer(c).key_hi;
                }
                above = M.above;
            } else if (by_mass) {
                key_lo = order_key(cut);
                ull m = 0, none;
                each([&](float v, int, int) { m += v > cut ? R.mass(v) : 0ull; });
                cluster_sum(m, 0, whole, none);
                whole += ties * R.mass(cut);
            }
            if (by_mass) limit = R.mass_limit(whole);
            while (true) {
                const uint32_t span = key_hi - key_lo;
                const int shift = span < S_RADIX ? 0 : 22 - __clz(span);
                csync();                       // the cluster has read the last step's histograms
                for (int i = tid; i < 4 * S_RADIX; i += THREADS) M.hist[i] = 0;
                if (tid == 0) M.best = -1;
                __syncthreads();
                each([&](float v, int, int) {
                    if (!(v > -INFINITY)) return;
                    const uint32_t key = order_key(v);
                    if (key < key_lo || key > key_hi) return;
                    const int b = (int) ((key_hi - key) >> shift);
                    const ull m = by_mass ? R.mass(v) : 1ull;
                    if (m == 0) return;
                    atomicAdd(&M.hist[b], (uint32_t) m & 0x7FFu);
                    if (by_mass) {
                        atomicAdd(&M.hist[S_RADIX + b], (uint32_t) (m >> 11) & 0x7FFu);
                        atomicAdd(&M.hist[2 * S_RADIX + b], (uint32_t) (m >> 22) & 0x7FFu);
                        atomicAdd(&M.hist[3 * S_RADIX + b], (uint32_t) (m >> 33));
                    }
                });
                csync();
                constexpr int PR = S_RADIX / THREADS;
                ull v[PR] = {}, sum = 0, t;
#pragma unroll
                for (int j = 0; j < PR; j++) {
                    for (int c = 0; c < C; c++) {
                        const uint32_t * h = peer(c).hist + PR * tid + j;
                        v[j] += (ull) h[0] + ((ull) h[S_RADIX] << 11) + ((ull) h[2 * S_RADIX] << 22) + ((ull) h[3 * S_RADIX] << 33);
                    }
                    sum += v[j];
                }
                ull run = above + block_scan<WARPS>(sum, M.scan, t) - sum, at[PR];
#pragma unroll
                for (int j = 0; j < PR; j++) {
                    at[j] = run;
                    if (v[j] && run <= limit) atomicMax(&M.best, PR * tid + j);
                    run += v[j];
                }
                __syncthreads();
                const int best = M.best;
#pragma unroll
                for (int j = 0; j < PR; j++)
                    if (PR * tid + j == best) M.above = at[j];
                __syncthreads();
                above = M.above;
                key_hi -= (uint32_t) best << shift;
                if (shift == 0) break;
                key_lo = max(key_lo, key_hi - ((1u << shift) - 1));
            }
            const float at = key_value(key_hi);
            const ull n = by_mass ? (limit - above) / R.mass(at) + 1 : limit - above + 1;
            ties = after_k && at == cut ? min(ties, n) : n;
            cut = at;
        }
    }

    // ---- the warps' masses, in order of index; then the token's warp is cut into WARPS parts, and the part's vectors
    const float w_cut = cut > -INFINITY ? (cut == top ? 1.0f : R.weight(cut)) : 0.0f;
    const ull m_cut = w_cut >= R.min_p ? mass_of(w_cut) : 0ull;
    auto vec_mass = [&](const uint4 & r, int & eq) {
        uint32_t hi = 0, lo = 0;
        if (ties) {
#pragma unroll
            for (int e = 0; e < E; e++) eq += vec16<T>::at(r, e) == cut;
        }
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float v[2] = { vec16<T>::at(r, e), vec16<T>::at(r, e + 1) };
            float2 w = R.weight2(R.distance2(v[0], v[1]));
            w.x = v[0] > cut && w.x >= R.min_p ? w.x : 0.0f;
            w.y = v[1] > cut && w.y >= R.min_p ? w.y : 0.0f;
            uint32_t h[2], l[2];
            mass_parts2(w, h, l);
            hi += h[0] + h[1];
            lo += l[0] + l[1];
        }
        return mass_sum(hi, lo, E);
    };
    int w0 = w_first, w1 = w0 + vecs;          // this warp's part of the row's vectors
    ull goal = 0, left = ties, total = 0;
    for (int level = 0; level < 2; level++) {
        ull m = 0;
        int eq = 0;
        const bool known = level == 0 && parts_known;
        if (!known) each_vec(w0, w1, [&](const uint4 & r, int) { m += vec_mass(r, eq); });
#pragma unroll
        for (int d = 16; d; d >>= 1) m += __shfl_xor_sync(0xFFFFFFFFu, m, d);
        eq = __reduce_add_sync(0xFFFFFFFFu, eq);
        __syncthreads();
        if (lane == 0 && !known) {
            M.part_mass[warp] = m;
            M.part_ties[warp] = eq;
        }
        if (level == 0) csync(); else __syncthreads();
        // part i of the row: warp i % WARPS of CTA i / WARPS, and then of the token's CTA only
        const int parts = level == 0 ? C * WARPS : WARPS;
        ull pm = 0, pe = 0, t;
        if (tid < parts) {
            const smem & Mc = level == 0 ? peer(tid / WARPS) : M;
            pm = Mc.part_mass[tid % WARPS];
            pe = Mc.part_ties[tid % WARPS];
            if (known) {
                const smem & M0 = peer(0);
                pm += M0.list_mass[0][tid] + ((ull) M0.list_mass[1][tid] << 14) + ((ull) M0.list_mass[2][tid] << 28);
                pe = M0.list_ties[tid];
            }
        }
        const ull ties_before = block_scan<WARPS>(pe, M.scan, t) - pe;
        const ull room = left > ties_before ? left - ties_before : 0;
        const ull mine = pm + min(room, pe) * m_cut;
        const ull run = block_scan<WARPS>(mine, M.scan, t);
        if (level == 0) {
            total = t;
            goal = R.goal(total);
        }
        if (goal >= run - mine && goal < run) {
            M.at = tid;
            M.goal = goal - (run - mine);
            M.ties = room;
        }
        if (level == 0) csync(); else __syncthreads();
        const int at = M.at;
        goal = M.goal;
        left = M.ties;
        if (level == 0) {
            if (at / WARPS != cta) return;     // the cluster has read what it needs
            w0 = at * vecs + (int) ((int64_t) warp * vecs / WARPS);
            w1 = at * vecs + (int) ((int64_t) (warp + 1) * vecs / WARPS);
        }
    }
    if (warp != M.at) return;
    for (int i = w0; i < w1; i++) {
        const int at = origin + i * 32 * E;
        const uint4 r = fetch(i);
        int eq = 0;
        const ull gt = vec_mass(r, eq);
        int eq_upto = eq;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xFFFFFFFFu, eq_upto, d);
            if (lane >= d) eq_upto += o;
        }
        ull room = left > (ull) (eq_upto - eq) ? left - (eq_upto - eq) : 0;
        const ull sum = gt + min(room, (ull) eq) * m_cut;
        ull upto = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const ull o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += o;
        }
        if (goal >= upto - sum && goal < upto) {
            ull run = upto - sum;
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float v = vec16<T>::at(r, e), w = v == cut ? w_cut : R.weight(v);
                ull m = 0;
                if (v > cut) {
                    m = w >= R.min_p ? mass_of(w) : 0ull;
                } else if (v == cut && room) {
                    room--;
                    m = m_cut;
                }
                if (m && goal >= run && goal < run + m) {
                    token[row] = at + e;
                    if (prob) prob[row] = R.prob(w, total);
                }
                run += m;
            }
        }
        const ull all = __shfl_sync(0xFFFFFFFFu, upto, 31);
        if (goal < all) return;
        goal -= all;
        const int eqs = __shfl_sync(0xFFFFFFFFu, eq_upto, 31);
        left = left > (ull) eqs ? left - eqs : 0;
    }
}

// ============================ host =========================================

bool paged_ok(const lnsb_paged_kv & a, int * st) {
    *st = LNSB_E_INVALID;
    const bool pow2 = a.page_size > 0 && (a.page_size & (a.page_size - 1)) == 0;
    if (a.type != LNSB_TYPE_F16 && a.type != LNSB_TYPE_BF16) return false;
    if (!pow2 || a.page_size < 8 || a.page_size > 1024) return false;
    if (a.head_dim != 16 && a.head_dim != 32 && a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256) return false;
    if (a.n_seqs < 0 || a.n_tokens < 0 || a.n_head_kv <= 0 || a.n_pages < 0 || a.table_ld < 0) return false;
    if (a.max_kv < 0 || a.max_kv > a.table_ld * a.page_size) return false;
    if (a.row_stride < a.head_dim || a.head_stride < a.head_dim || a.page_stride < a.head_dim) return false;
    if (a.page_stride % 8 || a.row_stride % 8 || a.head_stride % 8) return false;
    if ((reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache)) % 16) return false;
    if (a.n_tokens > 0 && a.n_seqs > 0 &&
        (a.k_cache == nullptr || a.v_cache == nullptr || a.page_table == nullptr || a.q_start == nullptr || a.kv_len == nullptr))
        return false;
    *st = LNSB_E_TOO_LARGE;
    if (a.max_kv > 0x7FFFFF00 || a.n_pages > 0x7FFFFFFF || a.n_tokens > 0x7FFFFFFF || a.n_seqs > 65536 || a.n_head_kv > 65535)
        return false;
    *st = 0;
    return true;
}
paged view_of(const lnsb_paged_kv & a) {
    paged P;
    P.table = a.page_table;
    P.q_start = a.q_start;
    P.kv_len = a.kv_len;
    P.table_ld = a.table_ld;
    P.n_pages = a.n_pages;
    P.n_tokens = a.n_tokens;
    P.max_kv = a.max_kv;
    P.page_stride = a.page_stride;
    P.row_stride = a.row_stride;
    P.head_stride = a.head_stride;
    P.n_seqs = a.n_seqs;
    P.page_shift = 31 - __builtin_clz((unsigned) a.page_size);
    P.n_head_kv = a.n_head_kv;
    return P;
}

template <class TI, class TC>
int launch_append(const lnsb_paged_append_args & a, cudaStream_t s) {
    const lnsb_paged_kv & c = a.kv;
    const TI * k = static_cast<const TI *>(a.k), * v = static_cast<const TI *>(a.v), * q = static_cast<const TI *>(a.q);
    TC * qo = static_cast<TC *>(a.q_out), * kc = static_cast<TC *>(c.k_cache), * vc = static_cast<TC *>(c.v_cache);
    const uintptr_t at = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(q) |
                         reinterpret_cast<uintptr_t>(qo) | reinterpret_cast<uintptr_t>(a.cos_sin);
    const int64_t ld = ((a.k_ld | a.v_ld | a.q_ld) * (int64_t) sizeof(TI)) | (a.q_out_ld * (int64_t) sizeof(TC));
    const bool neox = a.neox != 0;
    if (at % 16 == 0 && ld % 16 == 0 && a.n_dims % 16 == 0) {
        const int64_t per = (neox ? a.n_dims / 16 : a.n_dims / 8) + (c.head_dim - a.n_dims) / 8;
        const int64_t units = (a.n_head + c.n_head_kv) * per + (int64_t) c.n_head_kv * (c.head_dim / 8);
        // one thread a unit while that keeps a block within one token; short tokens share a block
        const int64_t tokens = std::max<int64_t>(1, std::min<int64_t>(256 / units, c.n_tokens));
        if (units > 0x7FFFFFFF / 2) return LNSB_E_TOO_LARGE;
        auto kern = neox ? k_paged_append_vec<TI, TC, true> : k_paged_append_vec<TI, TC, false>;
        launch_k(kern, dim3((unsigned) ((c.n_tokens + tokens - 1) / tokens)), dim3(256), 0, s, view_of(c), k, v, q, qo, a.cos_sin,
                 a.k_ld, a.v_ld, a.q_ld, a.q_out_ld, a.n_head, c.head_dim, a.n_dims, (int) tokens, kc, vc);
        return launch_status();
    }
    const int64_t per = a.n_dims / 2 + (c.head_dim - a.n_dims);
    const int64_t n = c.n_tokens * ((int64_t) (a.n_head + c.n_head_kv) * per + (int64_t) c.n_head_kv * c.head_dim);
    const int64_t blocks = std::min<int64_t>((n + 255) / 256, k_sms * 64);
    launch_k(k_paged_append<TI, TC>, dim3((unsigned) blocks), dim3(256), 0, s, view_of(c), k, v, q, qo, a.cos_sin, a.k_ld, a.v_ld,
             a.q_ld, a.q_out_ld, a.n_head, c.head_dim, a.n_dims, a.neox, kc, vc);
    return launch_status();
}

constexpr int k_max_devices = 64, k_smem_most = 227 * 1024;

// dynamic shared memory of a kernel, once per device
template <class K>
int allow_smem(K kern, bool (&done)[k_max_devices], int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int) e;
    if (dev < 0 || dev >= k_max_devices) return LNSB_E_NO_DEVICE;
    if (done[dev]) return 0;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return (int) e;
    done[dev] = true;
    return 0;
}

template <class T, int THREADS, bool HELD>
int launch_sample(const lnsb_sample_args & a, int C, int vecs, cudaStream_t s) {
    auto kern = k_sample<T, THREADS, HELD>;
    static bool attr[k_max_devices] = {};
    const int st = allow_smem(kern, attr, HELD ? k_smem_most : (int) sizeof(sample_smem));
    if (st != 0) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (a.n_rows * C));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = sizeof(sample_smem) + (HELD ? (size_t) vecs * THREADS * 16 : 0);
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = LNSB_PDL;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = { (unsigned) C, 1, 1 };
    cfg.attrs = at;
    cfg.numAttrs = HELD ? 2 : 1;
    (void) cudaLaunchKernelEx(&cfg, kern, static_cast<const T *>(a.logits), a.ld, (int) a.n_vocab, vecs, C, a.temperature, a.top_k,
                              a.top_p, a.min_p, a.u, a.token, a.prob);    // an error stays in cudaGetLastError
    return launch_status();
}
template <class T>
int launch_sample_rows(const lnsb_sample_args & a, cudaStream_t s) {
    constexpr int E = vec16<T>::N;
    const int need = (int) a.n_vocab + E - 1;                            // a row may start inside a vector
    auto vecs = [&](int threads, int C) { return (need + C * threads * E - 1) / (C * threads * E); };
    // few rows: as many CTAs to each as leave every one an SM of its own and its threads a vector each
    constexpr int threads = 512;
    int C = k_row_ctas;
    while (C > 1 && (a.n_rows * C > k_sms || need <= C / 2 * threads * E)) C /= 2;
    const int held = vecs(threads, C);
    if (a.n_rows <= k_sms && held * threads * E < 65536 && (int) sizeof(sample_smem) + held * threads * 16 <= k_smem_most)
        return launch_sample<T, threads, true>(a, C, held, s);
    // the row stays in memory: one to an SM, else two
    if (a.n_rows <= k_sms) return launch_sample<T, 1024, false>(a, 1, vecs(1024, 1), s);
    return launch_sample<T, 512, false>(a, 1, vecs(512, 1), s);
}

std::atomic<uint32_t> wait_limit{ k_wait_cycles };   // of lnsb_paged_attn's later calls

constexpr float k_log2e = 1.44269504088896340736f;

template <class T, int D>
int launch_rows(const lnsb_paged_attn_args & a, int64_t rows_most, cudaStream_t s) {
    auto kern = k_paged_attn_rows<T, D>;
    static bool attr[k_max_devices] = {};
    const int st = allow_smem(kern, attr, a_smem<D>());
    if (st != 0) return st;
    unsigned char * w = static_cast<unsigned char *>(a.work);
    launch_k(kern, dim3(A_CTAS), dim3(128), (size_t) a_smem<D>(), s, view_of(a.kv), static_cast<const T *>(a.q),
             static_cast<T *>(a.dst), static_cast<const T *>(a.kv.k_cache), static_cast<const T *>(a.kv.v_cache), a.q_ld,
             a.dst_ld, a.n_head / a.kv.n_head_kv, a.scale * k_log2e, a.window, rows_most, reinterpret_cast<int *>(w),
             reinterpret_cast<float *>(w + A_COUNT_BYTES));
    return launch_status();
}

using encode_fn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                               const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
encode_fn tensor_map_encoder() {
    static const encode_fn fn = [] {
        void * f = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) != cudaSuccess) f = nullptr;
        return reinterpret_cast<encode_fn>(f);
    }();
    return fn;
}
// a cache as (64 of dim, row of the page, kv head, page); false: not to be described
bool map_cache(CUtensorMap * m, const lnsb_paged_kv & c, void * cache, int keys) {
    const encode_fn encode = tensor_map_encoder();
    if (encode == nullptr) return false;
    const cuuint64_t dims[4] = { (cuuint64_t) c.head_dim, (cuuint64_t) c.page_size, (cuuint64_t) c.n_head_kv, (cuuint64_t) c.n_pages };
    const cuuint64_t strides[3] = { (cuuint64_t) c.row_stride * 2, (cuuint64_t) c.head_stride * 2, (cuuint64_t) c.page_stride * 2 };
    const cuuint32_t box[4] = { 64, (cuuint32_t) std::min(c.page_size, keys), 1, 1 }, one[4] = { 1, 1, 1, 1 };
    return encode(m, c.type == LNSB_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, cache, dims,
                  strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class T, int D>
int launch_attn_dim(const lnsb_paged_attn_args & a, cudaStream_t s) {
    if constexpr (D == 64 || D == 128) {
        const int G = a.n_head / a.kv.n_head_kv;
        CUtensorMap km, vm;
        // More than 16 rows go to the tiles: the rows kernel reads K and V again for every 16.  64 sequences over 4,096
        // rows, 8 kv heads of 128: 16 rows each 226 us by tiles and 189 by rows, 20 to 32 rows 227 and 346, 256 rows
        // 338 and 2,820; at head dim 64 (4 kv heads) 104 and 88, 105 and 146, 165 and 804.  (One sequence of 9 to 16 rows
        // leaves the rows kernel few warps to a key: 34 us by tiles and 67 by rows over 2,048 rows.  There the rule is wrong
        // by up to two times, and so at head dim 64 from 64 rows on, where one short sequence takes 40 by tiles, 33 by rows.)
        // scale > 0: the tiles take the maximum before the scale
        if (a.max_q > ROWS / G && a.kv.n_pages > 0 && a.scale > 0.0f && std::isfinite(a.scale) &&
            map_cache(&km, a.kv, a.kv.k_cache, b_keys<D>()) && map_cache(&vm, a.kv, a.kv.v_cache, b_keys<D>())) {
            auto kern = k_paged_attn_tiles<T, D>;
            static bool attr[k_max_devices] = {};
            int st = allow_smem(kern, attr, b_smem<D>());
            // sequences of few rows go to the rows kernel; one sequence alone does not split (which of several have
            // few is known on the device only: a launch without such rows ends at the plan)
            const bool both = a.kv.n_seqs > 1;
            if (st == 0 && both) st = launch_rows<T, D>(a, ROWS, s);
            if (st != 0) return st;
            tile_plan L;
            L.rows_above = both ? ROWS : 0;
            L.window = a.window;
            L.G = G;
            L.key_shift = D == 128 ? 7 : 6;
            static_assert(b_keys<D>() == (D == 128 ? 1 << 7 : 1 << 6), "keys of a tile");
            unsigned char * w = static_cast<unsigned char *>(a.work) + A_WORK;
            launch_k(kern, dim3(B_CTAS), dim3(B_THREADS), (size_t) b_smem<D>(), s, km, vm, view_of(a.kv), L,
                     static_cast<const T *>(a.q), static_cast<T *>(a.dst), a.q_ld, a.dst_ld, a.scale * k_log2e,
                     reinterpret_cast<int *>(w), reinterpret_cast<float *>(w + B_COUNT_BYTES),
                     wait_limit.load(), reinterpret_cast<unsigned long long *>(w + B_WORK));
            return launch_status();
        }
    }
    return launch_rows<T, D>(a, INT64_MAX, s);
}
template <class T>
int launch_attn(const lnsb_paged_attn_args & a, cudaStream_t s) {
    switch (a.kv.head_dim) {
        case 16:  return launch_attn_dim<T, 16>(a, s);
        case 32:  return launch_attn_dim<T, 32>(a, s);
        case 64:  return launch_attn_dim<T, 64>(a, s);
        case 128: return launch_attn_dim<T, 128>(a, s);
        default:  return launch_attn_dim<T, 256>(a, s);
    }
}

}  // namespace
}  // namespace lnsb

using namespace lnsb;

extern "C" {

int lnsb_paged_append(const lnsb_paged_append_args * a, lnsb_stream_t stream) {
    if (a == nullptr) return LNSB_E_INVALID;
    int st = 0;
    if (!paged_ok(a->kv, &st)) return st;
    const lnsb_paged_kv & c = a->kv;
    const int nh = a->q != nullptr ? a->n_head : 0;
    if ((a->q == nullptr) != (a->q_out == nullptr) || a->n_head < 0 || (a->q != nullptr && a->n_head == 0)) return LNSB_E_INVALID;
    if (a->n_dims < 0 || a->n_dims % 2 != 0 || a->n_dims > c.head_dim || (a->n_dims > 0 && a->cos_sin == nullptr))
        return LNSB_E_INVALID;
    if (a->in_type != LNSB_TYPE_F32 && a->in_type != LNSB_TYPE_F16 && a->in_type != LNSB_TYPE_BF16) return LNSB_E_INVALID;
    const int64_t kvw = (int64_t) c.n_head_kv * c.head_dim, qw = (int64_t) nh * c.head_dim;
    if (a->k_ld < kvw || a->v_ld < kvw || (nh > 0 && (a->q_ld < qw || a->q_out_ld < qw))) return LNSB_E_INVALID;
    if (c.n_tokens == 0 || c.n_seqs == 0) return 0;
    if (a->k == nullptr || a->v == nullptr) return LNSB_E_INVALID;
    lnsb_paged_append_args b = *a;
    b.n_head = nh;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool f16 = c.type == LNSB_TYPE_F16;
    switch (a->in_type) {
        case LNSB_TYPE_F32: return f16 ? launch_append<float, __half>(b, s) : launch_append<float, __nv_bfloat16>(b, s);
        case LNSB_TYPE_F16: return f16 ? launch_append<__half, __half>(b, s) : launch_append<__half, __nv_bfloat16>(b, s);
        default:            return f16 ? launch_append<__nv_bfloat16, __half>(b, s) : launch_append<__nv_bfloat16, __nv_bfloat16>(b, s);
    }
}

int64_t lnsb_paged_attn_work_bytes(void) { return WORK_BYTES; }

int lnsb_paged_attn_wait_limit(int64_t cycles) {
    if (cycles < 0) return LNSB_E_INVALID;
    wait_limit.store((uint32_t) std::min<int64_t>(cycles, k_wait_cycles));
    return 0;
}

int lnsb_paged_attn(const lnsb_paged_attn_args * a, lnsb_stream_t stream) {
    if (a == nullptr) return LNSB_E_INVALID;
    int st = 0;
    if (!paged_ok(a->kv, &st)) return st;
    const lnsb_paged_kv & c = a->kv;
    if (a->n_head <= 0 || a->n_head % c.n_head_kv != 0 || a->max_q < 0 || a->window < 0) return LNSB_E_INVALID;
    if (c.n_tokens * a->n_head > 0x7FFFFFFF) return LNSB_E_TOO_LARGE;
    const int64_t w = (int64_t) a->n_head * c.head_dim;
    if (a->q_ld < w || a->dst_ld < w || a->q_ld % 8 || a->dst_ld % 8) return LNSB_E_INVALID;
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->dst) | reinterpret_cast<uintptr_t>(a->work)) % 16)
        return LNSB_E_INVALID;
    if (c.n_tokens == 0 || c.n_seqs == 0) return 0;
    if (a->q == nullptr || a->dst == nullptr || a->work == nullptr || a->work_bytes < lnsb_paged_attn_work_bytes())
        return LNSB_E_INVALID;
    lnsb_paged_attn_args b = *a;
    if (b.window >= c.max_kv) b.window = 0;     // hides no row; the kernels' windows are below 2^31
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return c.type == LNSB_TYPE_F16 ? launch_attn<__half>(b, s) : launch_attn<__nv_bfloat16>(b, s);
}

int lnsb_paged_errors(int64_t * bad_pages, int64_t * timeouts) {
    // the device's counts only grow, also while they are read; what was handed out is kept here
    static std::mutex lock;
    static unsigned long long given[k_max_devices][2];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return (int) e;
    if (dev < 0 || dev >= k_max_devices) return LNSB_E_NO_DEVICE;
    const std::lock_guard<std::mutex> hold(lock);
    unsigned long long v[2] = {};
    e = cudaMemcpyFromSymbol(v, g_paged_errors, sizeof(v));
    if (e != cudaSuccess) return (int) e;
    for (int i = 0; i < 2; i++) {
        const unsigned long long before = v[i] < given[dev][i] ? 0 : given[dev][i];     // 0: the device was reset
        given[dev][i] = v[i];
        v[i] -= before;
    }
    if (bad_pages) *bad_pages = (int64_t) v[0];
    if (timeouts) *timeouts = (int64_t) v[1];
    return 0;
}

int lnsb_sample(const lnsb_sample_args * a, lnsb_stream_t stream) {
    if (a == nullptr || a->n_rows < 0 || a->n_vocab <= 0 || a->ld < a->n_vocab) return LNSB_E_INVALID;
    if (a->type != LNSB_TYPE_F32 && a->type != LNSB_TYPE_F16 && a->type != LNSB_TYPE_BF16) return LNSB_E_INVALID;
    if (a->n_rows == 0) return 0;
    if (a->logits == nullptr || a->u == nullptr || a->token == nullptr) return LNSB_E_INVALID;
    if (a->n_vocab > (1 << 20) || a->n_rows > 0x7FFFFFFF) return LNSB_E_TOO_LARGE;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a->type == LNSB_TYPE_F32) return launch_sample_rows<float>(*a, s);
    return a->type == LNSB_TYPE_F16 ? launch_sample_rows<__half>(*a, s) : launch_sample_rows<__nv_bfloat16>(*a, s);
}

}  // extern "C"
