// Shared pieces of the paged KV cache's kernels: which rows and keys a sequence has, the join of partial softmax
// results, and the small PTX wrappers both attention kernels use.
//
// A cache is two pools [n_pages, kv_heads, page_size, hd]: the rows of one page and head are contiguous, so a tile
// of keys is a few whole runs of page_size * hd elements.  Rows of a call are packed: row r of sequence b and K/V
// head g is new token r / group, query head g * group + r % group, so that all the query heads that share a K/V head
// read it together.
//
// The softmax runs in base 2 (scores times log2 e); m is the running maximum in those units, l the sum of
// 2^(s - m), acc the sum of 2^(s - m) v, all in 32 bits.  A row that sees no key has m = -inf and l = 0.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "common.hpp"

namespace qb {

// Sequences of at most this many packed rows go to the kernels for few rows, the others to the prompt kernel; calls of at
// most PG_FEW_IN_ALL rows a K/V head go to the former as a whole where that is little work (pg_rows_plan).
constexpr uint32_t PG_FEW_ROWS = 16, PG_FEW_IN_ALL = 1024;

constexpr float PG_LOG2E = 1.4426950408889634f, PG_LN2 = 0.6931471805599453f;

struct PgArgs {
    const void* q;              // [tokens, q_stride], head h at column h * hd
    const uint16_t* k;          // pools
    const uint16_t* v;
    const int32_t* table;       // [batch, table_stride] page numbers; the prefix phase: [width]
    const int32_t* kv_lens;     // [batch]
    const int32_t* cu_q;        // [batch + 1], or null: one token per sequence
    const int32_t* prefix_lens; // [batch], or null
    const float* slopes;        // [heads], or null
    int32_t* status;
    uint64_t q_stride, table_stride;
    uint32_t n_pages, ps_log, width;  // page size = 1 << ps_log; width: pages a table row can hold
    uint32_t batch, tokens, group, kv_heads;
    uint32_t causal;
    uint32_t shared;            // keys of a shared prefix: all tokens of the batch are one sequence that sees keys [0, shared)
    float score_mul;            // log2 e * scale without a cap; scale / cap with one
    float cap_mul;              // cap * log2 e, 0: no cap
    // results: rows of `out` [tokens, heads * hd], joined with the state that a first phase left of every row
    uint16_t* out;
    float* lse;                 // [tokens, heads] or null
    const float* base_acc;      // [tokens * heads][hd] and [tokens * heads][2] (m, l), or null
    const float* base_ml;
    float* rows_acc;            // the same two, written instead of out by a first phase
    float* rows_ml;
    float* parts;               // partial results of units that several CTAs share
    int32_t* meta;
};

struct PgSeq {
    uint32_t q0, q_len, kv;  // rows [q0, q0 + q_len) of the batch; keys [0, kv)
    uint32_t prefix;         // keys that every row sees
};

__device__ __forceinline__ void pg_report(int32_t* status, int32_t code) { atomicCAS(status, 0, code); }

// What sequence b of the call has; lengths that do not fit the call are cut and reported.
__device__ __forceinline__ PgSeq pg_seq(const PgArgs& a, uint32_t b) {
    PgSeq s;
    if (a.shared) {
        int32_t n = a.cu_q ? a.cu_q[a.batch] : (int32_t)a.tokens;
        s.q0 = 0;
        s.q_len = n < 0 ? 0u : min((uint32_t)n, a.tokens);
        s.kv = a.shared;
        s.prefix = a.shared;
        return s;
    }
    int32_t lo = (int32_t)b, hi = lo + 1, kv = a.kv_lens[b];
    if (a.cu_q) {
        lo = a.cu_q[b];
        hi = a.cu_q[b + 1];
    }
    const int64_t room = (int64_t)a.width << a.ps_log;
    if (lo < 0 || hi < lo || hi > (int32_t)a.tokens || kv < 0 || kv > room) {
        pg_report(a.status, QB200_ERR_LENGTH);
        lo = max(0, min(lo, (int32_t)a.tokens));
        hi = max(lo, min(hi, (int32_t)a.tokens));
        kv = kv < 0 ? 0 : (int32_t)(kv > room ? room : kv);
    }
    s.q0 = (uint32_t)lo;
    s.q_len = (uint32_t)(hi - lo);
    s.kv = (uint32_t)kv;
    const int32_t p = a.prefix_lens ? a.prefix_lens[b] : 0;
    s.prefix = a.causal ? (uint32_t)max(p, 0) : 0xFFFFFFFFu;
    return s;
}

// Keys that token i of the sequence sees: its position is kv - q_len + i (negative for a sequence with fewer keys
// than new tokens, whose first tokens see nothing).
__device__ __forceinline__ uint32_t pg_limit(const PgSeq& s, uint32_t i) {
    const int32_t to = (int32_t)s.kv - (int32_t)s.q_len + (int32_t)i + 1;
    return min(s.kv, max((uint32_t)max(to, 0), s.prefix));
}

// Position of token i, counted from the first key that this phase reads (the bias by distance counts from it).
__device__ __forceinline__ int32_t pg_position(const PgArgs& a, const PgSeq& s, uint32_t i) {
    if (!a.shared) return (int32_t)s.kv - (int32_t)s.q_len + (int32_t)i;
    // the prefix phase: row i is token i of the whole batch; its sequence's own keys follow the prefix
    uint32_t b = i;
    int32_t lo = (int32_t)i, hi = lo + 1;
    if (a.cu_q) {
        uint32_t l = 0, r = a.batch;  // the last b with cu_q[b] <= i
        while (r - l > 1) {
            const uint32_t mid = (l + r) >> 1;
            if (a.cu_q[mid] <= (int32_t)i) l = mid; else r = mid;
        }
        b = l;
        lo = a.cu_q[b];
        hi = a.cu_q[b + 1];
    }
    const int64_t room = (int64_t)0x7FFFFFFF - a.shared;
    return (int32_t)a.shared + (int32_t)min((int64_t)max(a.kv_lens[b], 0), room) - (hi - lo) + ((int32_t)i - lo);
}

// 2^x, flushing far below the range to zero.
__device__ __forceinline__ float pg_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pg_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// cap * log2 e * tanh(x), with an error relative to the result: a cap far above the scores leaves them as they are, so an
// error in units of the cap would not do (1e5: scores off by 0.01).  Below 0.3 x times the polynomial in x^2 of the least
// relative error there (1.3e-8, fitted by reweighted least squares); above, 1 - 2 / (e^(2x) + 1), which errs by a few
// 2^-24 (e^(2x) = 0 and inf give -1 and 1).  (tanh.approx errs by 2^-11.)
__device__ __forceinline__ float pg_cap(float x, float cap_mul) {
    const float e = pg_exp2(x * (2.0f * PG_LOG2E)), u = x * x;
    const float far = fmaf(-2.0f * cap_mul, pg_rcp(e + 1.0f), cap_mul);
    const float near = cap_mul * x * fmaf(u, fmaf(u, fmaf(u, -0.0503677242f, 0.133148476f), -0.333330601f), 1.0f);
    return fabsf(x) <= 0.3f ? near : far;
}

template <typename T> struct PgType;
template <> struct PgType<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ float widen(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
    static __device__ __forceinline__ float2 widen2(uint32_t b) { return make_float2(__uint_as_float(b << 16), __uint_as_float(b & 0xFFFF0000u)); }
};
template <> struct PgType<__half> {
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    }
    static __device__ __forceinline__ float widen(uint16_t b) { return __half2float(__ushort_as_half(b)); }
    static __device__ __forceinline__ float2 widen2(uint32_t b) { return make_float2(widen((uint16_t)(b & 0xFFFFu)), widen((uint16_t)(b >> 16))); }
};

// Weight of a state with maximum m against the joint maximum M (a state without keys has none).
__device__ __forceinline__ float pg_weight(float m, float M) { return m == -INFINITY ? 0.0f : pg_exp2(m - M); }

// The end of one row's state (m, l): joined with what an earlier phase left and normalised, or kept for a later phase.
// acc goes through pg_store4, four columns at a time.
struct PgEnd {
    float f, g;  // factors of this state's acc and of the earlier phase's (1 / l is in both)
    uint32_t row;
};
__device__ __forceinline__ PgEnd pg_end(const PgArgs& a, uint32_t token, uint32_t head, float m, float l, bool first) {
    PgEnd e = {1.0f, 0.0f, token * a.group * a.kv_heads + head};
    if (a.rows_acc) {
        if (first) *reinterpret_cast<float2*>(a.rows_ml + (uint64_t)e.row * 2) = make_float2(m, l);
        return e;
    }
    if (a.base_acc) {
        const float2 ml = *(reinterpret_cast<const float2*>(a.base_ml) + e.row);
        const float M = fmaxf(m, ml.x);
        e.f = pg_weight(m, M);
        e.g = pg_weight(ml.x, M);
        l = fmaf(l, e.f, ml.y * e.g);
        m = M;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    e.f *= inv;
    e.g *= inv;
    if (a.lse && first) a.lse[e.row] = l == 0.0f ? -INFINITY : (m + log2f(l)) * PG_LN2;
    return e;
}
template <typename T, uint32_t HD>
__device__ __forceinline__ void pg_store4(const PgArgs& a, const PgEnd& e, uint32_t col, float4 v) {
    if (a.rows_acc) {
        *reinterpret_cast<float4*>(a.rows_acc + (uint64_t)e.row * HD + col) = v;
        return;
    }
    v.x *= e.f;
    v.y *= e.f;
    v.z *= e.f;
    v.w *= e.f;
    if (a.base_acc) {
        const float4 w = *reinterpret_cast<const float4*>(a.base_acc + (uint64_t)e.row * HD + col);
        v.x = fmaf(w.x, e.g, v.x);
        v.y = fmaf(w.y, e.g, v.y);
        v.z = fmaf(w.z, e.g, v.z);
        v.w = fmaf(w.w, e.g, v.w);
    }
    uint2 o;
    o.x = PgType<T>::pack(v.x, v.y);
    o.y = PgType<T>::pack(v.z, v.w);
    *reinterpret_cast<uint2*>(a.out + (uint64_t)e.row * HD + col) = o;
}
template <typename T, uint32_t HD>
__device__ __forceinline__ void pg_emit(const PgArgs& a, uint32_t token, uint32_t head, uint32_t col, float m, float l, float4 v) {
    pg_store4<T, HD>(a, pg_end(a, token, head, m, l, col == 0), col, v);
}

qb200_status pg_sms(uint32_t* n);  // SMs of the current device
uint32_t pg_spin_limit();          // polls of a wait inside the prompt kernel
// Attention for few rows (paged_rows.cu): how it runs and the floats of partial results that takes.
struct PgRows {
    bool units;      // a cluster of 2^c_log CTAs per unit of 16 rows, row_tiles of them a sequence and K/V head; otherwise equal runs of all tiles, and a second kernel
    uint32_t c_log, grid, row_tiles;
    uint64_t floats;
};
uint64_t pg_rows_most_tiles(const PgArgs& a);  // below 2^32, or the call is refused
PgRows pg_rows_plan(const PgArgs& a, uint32_t hd, uint32_t sms, uint32_t row_tiles);
qb200_status pg_rows_launch(const PgArgs& a, int dtype, uint32_t hd, const PgRows& how, cudaStream_t st);
// Attention for many rows (paged_prompt.cu): over how many ranges a unit's keys are cut, the floats of partial results
// that takes, and the launch; min_rows: sequences of fewer packed rows are not its own.
uint32_t pg_prompt_splits(const PgArgs& a, uint32_t sms);
uint64_t pg_prompt_part_floats(const PgArgs& a, uint32_t splits, uint32_t hd);
qb200_status pg_prompt_launch(const PgArgs& a, int dtype, uint32_t hd, uint32_t splits, uint32_t min_rows, cudaStream_t st);

// Launches with programmatic stream serialization (see the kernels' first lines), in clusters of `cluster` CTAs.
template <typename... KArgs, typename... Args>
static cudaError_t pg_launch_cluster(void (*kernel)(KArgs...), dim3 grid, dim3 block, uint32_t smem, cudaStream_t st, uint32_t cluster, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}
template <typename... KArgs, typename... Args>
static cudaError_t pg_launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, uint32_t smem, cudaStream_t st, Args... args) {
    return pg_launch_cluster(kernel, grid, block, smem, st, 1, args...);
}

}  // namespace qb
