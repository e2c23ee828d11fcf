// The paged KV cache's entry points and the append kernel.
//
// Append is bounded by bytes (latency when few tokens arrive): every element of q, k and v is read once and written
// once (8620 tokens, 32 / 8 heads of 128, bf16: 38 us, 5.7 TB/s, 0.87 of measured; 16 tokens: 2.4 us in a graph).  A
// block takes one token; a thread keeps its eight pairs of angles in registers and walks the heads with them, 16
// elements (two 16-byte groups, the halves of the rotated pairs) at a time, two heads in flight (three: 39.9 us).
#include <atomic>
#include <cmath>
#include <string>

#include "paged.cuh"

namespace qb {

struct AppendArgs {
    const void *q, *k, *v;
    uint64_t q_stride, k_stride, v_stride, table_stride, n_pos;
    const float *cosv, *sinv;
    const int32_t *positions, *table, *kv_lens, *cu_q;
    uint16_t *q_out, *kp, *vp;
    int32_t* status;
    uint32_t heads, kv_heads, hd, rot, batch, tokens, n_pages, ps_log, width;
};

template <typename X> __device__ __forceinline__ void ap_load8(const X* p, float (&r)[8]);
template <> __device__ __forceinline__ void ap_load8<float>(const float* p, float (&r)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    r[0] = a.x; r[1] = a.y; r[2] = a.z; r[3] = a.w; r[4] = b.x; r[5] = b.y; r[6] = b.z; r[7] = b.w;
}
template <typename X> __device__ __forceinline__ void ap_load8(const X* p, float (&r)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        r[2 * i] = PgType<X>::widen((uint16_t)(w[i] & 0xFFFFu));
        r[2 * i + 1] = PgType<X>::widen((uint16_t)(w[i] >> 16));
    }
}
__device__ __forceinline__ float ap_load1(const float* p) { return *p; }
__device__ __forceinline__ float ap_load1(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float ap_load1(const __half* p) { return __half2float(*p); }
template <typename T> __device__ __forceinline__ void ap_store8(uint16_t* p, const float (&r)[8]) {
    uint4 o;
    o.x = PgType<T>::pack(r[0], r[1]);
    o.y = PgType<T>::pack(r[2], r[3]);
    o.z = PgType<T>::pack(r[4], r[5]);
    o.w = PgType<T>::pack(r[6], r[7]);
    *reinterpret_cast<uint4*>(p) = o;
}

// The rotation of one pair, the same bits in both forms of the kernel (which product is fused is not left to the compiler).
__device__ __forceinline__ void ap_turn(float& u, float& w, float c, float s) {
    const float p = u, r = w;
    u = fmaf(p, c, -__fmul_rn(r, s));
    w = fmaf(r, c, __fmul_rn(p, s));
}

// VEC: 16-byte aligned rows and a rotated width that is a multiple of 16; otherwise one pair of elements at a time.
template <typename X, typename T, bool VEC>
__global__ void __launch_bounds__(128) k_paged_append(const AppendArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t t = blockIdx.x, tid = threadIdx.x;
    // the token's sequence: how many of cu_q[1 .. batch] are at or below t
    uint32_t b = t;
    int32_t lo = (int32_t)t, hi = lo + 1;
    if (a.cu_q) {
        b = 0;
        for (uint32_t i0 = 0; i0 < a.batch; i0 += 128) {
            const uint32_t i = i0 + tid;
            b += (uint32_t)__syncthreads_count(i < a.batch && a.cu_q[i + 1] <= (int32_t)t);
        }
        if (b >= a.batch) return;  // a row behind the last sequence
        lo = a.cu_q[b];
        hi = a.cu_q[b + 1];
        if (b == 0 && (int32_t)t < lo && lo <= hi && hi <= (int32_t)a.tokens) return;  // a row before the first sequence
    }
    const int32_t kv = a.kv_lens[b];
    // (a 32-bit kv and hi - lo in [1, tokens]: no overflow in 64 bits)
    const int64_t place = (int64_t)kv - hi + (int64_t)t;
    bool write = place >= 0;
    int32_t page = 0;
    if (lo > (int32_t)t || hi <= (int32_t)t || lo < 0 || hi > (int32_t)a.tokens || kv < 0 || (place >= 0 && (place >> a.ps_log) >= a.width)) {
        if (tid == 0) pg_report(a.status, QB200_ERR_LENGTH);
        write = false;
    }
    if (write) {
        page = a.table[(uint64_t)b * a.table_stride + (uint64_t)(place >> a.ps_log)];
        if ((uint32_t)page >= a.n_pages) {
            if (tid == 0) pg_report(a.status, QB200_ERR_INVALID_PARAM);
            write = false;
        }
    }
    int64_t pos = a.positions ? (int64_t)a.positions[t] : place;
    if (pos < 0 || pos >= (int64_t)a.n_pos) {
        if (tid == 0 && (a.positions || place >= 0)) pg_report(a.status, QB200_ERR_INVALID_PARAM);
        pos = (int64_t)a.n_pos - 1;
    }
    const uint32_t half = a.rot >> 1, kv_end = a.heads + a.kv_heads, all = kv_end + a.kv_heads;
    const float *cp = a.cosv + (uint64_t)pos * half, *sp = a.sinv + (uint64_t)pos * half;
    const uint64_t in_page = (uint64_t)(place & ((1 << a.ps_log) - 1)) * a.hd;
    // head h of q | k | v: where it comes from and goes to (null: nowhere)
    auto from = [&](uint32_t h) -> const X* {
        if (h < a.heads) return static_cast<const X*>(a.q) + t * a.q_stride + (uint64_t)h * a.hd;
        if (h < kv_end) return static_cast<const X*>(a.k) + t * a.k_stride + (uint64_t)(h - a.heads) * a.hd;
        return static_cast<const X*>(a.v) + t * a.v_stride + (uint64_t)(h - kv_end) * a.hd;
    };
    auto to = [&](uint32_t h) -> uint16_t* {
        if (h < a.heads) return a.q_out + ((uint64_t)t * a.heads + h) * a.hd;
        if (!write) return nullptr;
        const uint32_t g = h < kv_end ? h - a.heads : h - kv_end;
        const uint64_t at = (((uint64_t)(uint32_t)page * a.kv_heads + g) << a.ps_log) * a.hd + in_page;
        return (h < kv_end ? a.kp : a.vp) + at;
    };
    if constexpr (VEC) {
        const uint32_t per = a.hd >> 4, j = tid % per, step = (128 / per) * gridDim.y;
        const bool turned = j * 16 < a.rot;
        float c[8], s[8];
        if (turned) {
            ap_load8(cp + j * 8, c);
            ap_load8(sp + j * 8, s);
        }
#pragma unroll 2
        for (uint32_t h = blockIdx.y * (128 / per) + tid / per; h < all; h += step) {
            const X* x = from(h);
            uint16_t* y = to(h);
            const bool turn = turned && h < kv_end;
            const uint32_t c0 = turn ? j * 8 : j * 16, c1 = turn ? half + j * 8 : j * 16 + 8;
            float u[8], w[8];
            ap_load8(x + c0, u);
            ap_load8(x + c1, w);
            if (turn) {
#pragma unroll
                for (int i = 0; i < 8; i++) ap_turn(u[i], w[i], c[i], s[i]);
            }
            if (y) {
                ap_store8<T>(y + c0, u);
                ap_store8<T>(y + c1, w);
            }
        }
    } else {
        const uint32_t pairs = a.hd >> 1;
        for (uint32_t i = blockIdx.y * 128 + tid; i < all * pairs; i += gridDim.y * 128) {
            const uint32_t h = i / pairs, j = i % pairs;
            const X* x = from(h);
            uint16_t* y = to(h);
            const bool turn = j < half && h < kv_end;
            // q and k: the pairs (j, rot / 2 + j) are rotated, the columns behind them go two by two, as v's do
            const uint32_t d0 = turn ? j : 2 * j, d1 = turn ? half + j : 2 * j + 1;
            float u = ap_load1(x + d0), w = ap_load1(x + d1);
            if (turn) ap_turn(u, w, cp[j], sp[j]);
            if (y) {
                const uint32_t o = PgType<T>::pack(u, w);
                y[d0] = (uint16_t)(o & 0xFFFFu);
                y[d1] = (uint16_t)(o >> 16);
            }
        }
    }
}

}  // namespace qb

namespace qb {

static bool pg_aligned(const void* p, uint64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// What every entry point asks of the cache and the batch.
static qb200_status pg_check_cache(const char* who, const qb200_paged_kv* kv, const qb200_paged_batch* b, uint64_t tokens) {
    const std::string w(who);
    if (!kv || !b) return fail(QB200_ERR_INVALID_PARAM, w + ": null cache or batch");
    if (!kv->k_pages || !kv->v_pages || !kv->status_dev) return fail(QB200_ERR_INVALID_PARAM, w + ": null pointer in the cache");
    if (!pg_aligned(kv->k_pages, 16) || !pg_aligned(kv->v_pages, 16)) return fail(QB200_ERR_INVALID_PARAM, w + ": the pools must be 16-byte aligned");
    if (kv->dtype != QB200_BF16 && kv->dtype != QB200_F16) return fail(QB200_ERR_NOT_SUPPORTED, w + ": a cache holds bf16 or f16");
    if (kv->head_dim != 64 && kv->head_dim != 128)
        return fail(QB200_ERR_NOT_SUPPORTED, w + ": head dim 64 or 128, got " + std::to_string(kv->head_dim));
    const uint32_t ps = kv->page_size;
    if (ps < 16 || ps > 256 || (ps & (ps - 1))) return fail(QB200_ERR_NOT_SUPPORTED, w + ": page size 16, 32, 64, 128 or 256, got " + std::to_string(ps));
    if (kv->kv_heads == 0 || kv->kv_heads > 65535) return fail(QB200_ERR_INVALID_PARAM, w + ": 1 .. 65535 K/V heads");
    if (kv->n_pages == 0 || kv->n_pages > 0x7FFFFFFFull) return fail(QB200_ERR_INVALID_PARAM, w + ": 1 .. 2^31 - 1 pages");
    if (!b->table || !b->kv_lens) return fail(QB200_ERR_INVALID_PARAM, w + ": null pointer in the batch");
    if (b->batch == 0 || b->batch > 0x7FFFFFFu) return fail(QB200_ERR_INVALID_PARAM, w + ": 1 .. 2^27 sequences");
    if (b->table_width == 0 || b->table_stride < b->table_width) return fail(QB200_ERR_LENGTH, w + ": table rows overlap or are empty");
    if ((uint64_t)b->table_width * ps > 0x7FFFFFFFull) return fail(QB200_ERR_NOT_SUPPORTED, w + ": a table row holds 2^31 keys or more");
    if (tokens > 0x7FFFFFFull) return fail(QB200_ERR_NOT_SUPPORTED, w + ": more than 2^27 new tokens");
    if ((uint64_t)b->batch * kv->kv_heads * (((uint64_t)b->table_width * ps + 63) / 64) > 0xFFFFFFFFull)
        return fail(QB200_ERR_NOT_SUPPORTED, w + ": the table spans 2^32 tiles of 64 keys or more");
    if (!b->cu_q && tokens != b->batch)
        return fail(QB200_ERR_LENGTH, w + ": without cu_q every sequence has one new token: " + std::to_string(tokens) + " tokens for " +
                                          std::to_string(b->batch) + " sequences");
    return QB200_OK;
}

static qb200_status pg_check_heads(const char* who, const qb200_paged_kv* kv, uint64_t tokens, uint32_t heads) {
    const std::string w(who);
    if (heads == 0 || heads % kv->kv_heads)
        return fail(QB200_ERR_INVALID_PARAM, w + ": " + std::to_string(heads) + " heads are no multiple of " + std::to_string(kv->kv_heads) + " K/V heads");
    if (tokens * heads > 0x7FFFFFFFull) return fail(QB200_ERR_NOT_SUPPORTED, w + ": 2^31 query rows or more");
    return QB200_OK;
}

static qb200_status pg_check_prefix(const char* who, const qb200_paged_kv* kv, const qb200_paged_batch* b, uint64_t prefix_len) {
    const std::string w(who);
    if (prefix_len == 0) return fail(QB200_ERR_INVALID_PARAM, w + ": no prefix (call qb200_paged_attention)");
    if (prefix_len > 0x7FFFFFFFull || prefix_len + (uint64_t)b->table_width * kv->page_size > 0x7FFFFFFFull)
        return fail(QB200_ERR_NOT_SUPPORTED, w + ": 2^31 keys or more");
    if (kv->kv_heads * ((prefix_len + 63) / 64) > 0xFFFFFFFFull) return fail(QB200_ERR_NOT_SUPPORTED, w + ": the prefix spans 2^32 tiles of 64 keys or more");
    return QB200_OK;
}

static qb200_status pg_check_attention(const char* who, const qb200_paged_kv* kv, const qb200_paged_batch* b, const void* q, uint64_t q_stride,
                                       uint64_t tokens, uint32_t heads, float scale, float softcap, const float* scratch, const void* out) {
    qb200_status st = pg_check_cache(who, kv, b, tokens);
    if (st) return st;
    const std::string w(who);
    if (tokens && (!q || !out)) return fail(QB200_ERR_INVALID_PARAM, w + ": null pointer");
    if ((st = pg_check_heads(who, kv, tokens, heads))) return st;
    if (q_stride < (uint64_t)heads * kv->head_dim || q_stride % 8) return fail(QB200_ERR_LENGTH, w + ": q's row stride must be a multiple of 8 that holds all heads");
    if (!pg_aligned(q, 16) || !pg_aligned(out, 16) || !pg_aligned(scratch, 16))
        return fail(QB200_ERR_INVALID_PARAM, w + ": q, out and scratch must be 16-byte aligned");
    if (!std::isfinite(scale) || !std::isfinite(softcap) || (softcap != 0.0f && softcap < 1e-6f))
        return fail(QB200_ERR_INVALID_PARAM, w + ": the scale must be finite, and the cap finite and 0 or at least 1e-6");
    if (tokens && q == out) return fail(QB200_ERR_INVALID_PARAM, w + ": the output must not overlap q");
    return QB200_OK;
}

static PgArgs pg_args(const qb200_paged_kv* kv, const qb200_paged_batch* b, uint64_t tokens, uint32_t heads) {
    PgArgs a = {};
    a.k = static_cast<const uint16_t*>(kv->k_pages);
    a.v = static_cast<const uint16_t*>(kv->v_pages);
    a.table = b->table;
    a.kv_lens = b->kv_lens;
    a.cu_q = b->cu_q;
    a.status = kv->status_dev;
    a.table_stride = b->table_stride;
    a.n_pages = (uint32_t)kv->n_pages;
    while ((1u << a.ps_log) < kv->page_size) a.ps_log++;
    a.width = b->table_width;
    a.batch = b->batch;
    a.tokens = (uint32_t)tokens;
    a.kv_heads = kv->kv_heads;
    a.group = heads / kv->kv_heads;
    a.causal = 1;
    return a;
}

qb200_status pg_sms(uint32_t* n) {
    static int count[64] = {};
    int dev = 0;
    QB_CUDA_TRY(cudaGetDevice(&dev));
    if (!count[dev & 63]) QB_CUDA_TRY(cudaDeviceGetAttribute(&count[dev & 63], cudaDevAttrMultiProcessorCount, dev));
    *n = (uint32_t)count[dev & 63];
    return QB200_OK;
}

static std::atomic<uint32_t> g_pg_spin_limit{4u << 20};
uint32_t pg_spin_limit() { return g_pg_spin_limit.load(std::memory_order_relaxed); }

// Which kernels a phase needs: sequences of at most PG_FEW_ROWS packed rows go to one, all others to the other; where
// only the device knows the lengths, both are launched.
struct PgPlan {
    bool few, many;
    uint32_t min_rows, splits;
    PgRows rows;
    uint64_t floats;  // scratch: the kernels follow one another and share it
};
static PgPlan pg_plan(const PgArgs& a, uint32_t hd, uint32_t sms) {
    PgPlan p = {};
    const uint64_t most = a.shared || a.cu_q ? (uint64_t)a.tokens * a.group : a.group;
    p.many = most > PG_FEW_ROWS;
    if (p.many && most <= PG_FEW_IN_ALL) {
        p.rows = pg_rows_plan(a, hd, sms, (uint32_t)div_ceil(most, PG_FEW_ROWS));
        if (p.rows.units) {
            p.few = true;
            p.many = false;
            return p;
        }
    }
    p.few = !p.many || (!a.shared && a.cu_q && a.group <= PG_FEW_ROWS);
    p.min_rows = p.few ? PG_FEW_ROWS + 1 : 1;
    if (p.few) {
        p.rows = pg_rows_plan(a, hd, sms, 1);
        p.floats = p.rows.floats;
    }
    if (p.many) {
        p.splits = pg_prompt_splits(a, sms);
        const uint64_t n = pg_prompt_part_floats(a, p.splits, hd);
        if (n > p.floats) p.floats = n;
    }
    p.floats = (p.floats + 3) / 4 * 4;
    return p;
}

static qb200_status pg_phase(const char* who, PgArgs a, int dtype, uint32_t hd, uint32_t sms, float* scratch, cudaStream_t st) {
    const PgPlan p = pg_plan(a, hd, sms);
    if (p.floats && !scratch) return fail(QB200_ERR_INVALID_PARAM, std::string(who) + ": the call needs its scratch");
    if (p.many) {
        a.parts = scratch;
        const qb200_status r = pg_prompt_launch(a, dtype, hd, p.splits, p.min_rows, st);
        if (r) return r;
    }
    if (p.few) {
        a.meta = reinterpret_cast<int32_t*>(scratch);
        a.parts = scratch + (uint64_t)p.rows.grid * 8;
        return pg_rows_launch(a, dtype, hd, p.rows, st);
    }
    return QB200_OK;
}

static void pg_scores(PgArgs& a, float scale, float softcap, const float* slopes) {
    // cap * log2 e and scale / cap leave the range of 32 bits for the largest caps, which do nothing: past 1e30 the cap takes less
    // than half a step from any score below 1e26
    if (softcap > 1e30f) softcap = 0.0f;
    a.score_mul = softcap > 0.0f ? scale / softcap : scale * PG_LOG2E;
    a.cap_mul = softcap > 0.0f ? softcap * PG_LOG2E : 0.0f;
    a.slopes = slopes;
}

template <typename X, typename T>
static cudaError_t launch_append(const AppendArgs& a, bool vec, dim3 grid, cudaStream_t st) {
    return vec ? pg_launch(k_paged_append<X, T, true>, grid, dim3(128), 0, st, a) : pg_launch(k_paged_append<X, T, false>, grid, dim3(128), 0, st, a);
}

}  // namespace qb

using namespace qb;

extern "C" {

qb200_status qb200_paged_rope_append(const qb200_paged_kv* kv, const qb200_paged_batch* batch, const void* q, const void* k, const void* v,
                                     int32_t x_dtype, uint64_t q_stride, uint64_t k_stride, uint64_t v_stride, uint64_t tokens, uint32_t heads,
                                     const float* cos, const float* sin, uint32_t rot_dim, uint64_t n_pos, const int32_t* positions,
                                     void* q_out, void* stream) {
    const char* who = "qb200_paged_rope_append";
    const std::string w(who);
    qb200_status st = pg_check_cache(who, kv, batch, tokens);
    if (st) return st;
    const uint32_t hd = kv->head_dim;
    if (x_dtype != QB200_F32 && x_dtype != QB200_BF16 && x_dtype != QB200_F16) return fail(QB200_ERR_NOT_SUPPORTED, w + ": f32, bf16 or f16 inputs");
    if (tokens == 0) return QB200_OK;
    if (!k || !v || !cos || !sin || (heads && (!q || !q_out))) return fail(QB200_ERR_INVALID_PARAM, w + ": null pointer");
    if (rot_dim == 0 || rot_dim > hd || (rot_dim & 1))
        return fail(QB200_ERR_INVALID_PARAM, w + ": the rotated width must be even and at most the head dim, got " + std::to_string(rot_dim));
    if (n_pos == 0 || n_pos > 0x7FFFFFFFull) return fail(QB200_ERR_INVALID_PARAM, w + ": 1 .. 2^31 - 1 rows of angles");
    const uint64_t esz = x_dtype == QB200_F32 ? 4 : 2;
    const uint64_t kw = (uint64_t)kv->kv_heads * hd, qw = (uint64_t)heads * hd;
    if ((heads && q_stride < qw) || k_stride < kw || v_stride < kw) return fail(QB200_ERR_LENGTH, w + ": rows overlap (a stride below heads * head_dim)");
    if (heads > 0xFFFFFu || (heads && !pg_aligned(q_out, 16)) || !pg_aligned(q, esz) || !pg_aligned(k, esz) || !pg_aligned(v, esz))
        return fail(QB200_ERR_INVALID_PARAM, w + ": q_out must be 16-byte aligned, inputs aligned to their elements");
    AppendArgs a = {};
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.table_stride = batch->table_stride;
    a.n_pos = n_pos;
    a.cosv = cos;
    a.sinv = sin;
    a.positions = positions;
    a.table = batch->table;
    a.kv_lens = batch->kv_lens;
    a.cu_q = batch->cu_q;
    a.q_out = static_cast<uint16_t*>(q_out);
    a.kp = static_cast<uint16_t*>(kv->k_pages);
    a.vp = static_cast<uint16_t*>(kv->v_pages);
    a.status = kv->status_dev;
    a.heads = heads;
    a.kv_heads = kv->kv_heads;
    a.hd = hd;
    a.rot = rot_dim;
    a.batch = batch->batch;
    a.tokens = (uint32_t)tokens;
    a.n_pages = (uint32_t)kv->n_pages;
    while ((1u << a.ps_log) < kv->page_size) a.ps_log++;
    a.width = batch->table_width;
    const bool vec = rot_dim % 16 == 0 && pg_aligned(cos, 16) && pg_aligned(sin, 16) && pg_aligned(k, 16) && pg_aligned(v, 16) && pg_aligned(q, 16) &&
                     (k_stride * esz) % 16 == 0 && (v_stride * esz) % 16 == 0 && (!heads || (q_stride * esz) % 16 == 0);
    // few tokens: the heads of a token over several blocks (one pass of a block's head lanes each)
    uint32_t sms = 0;
    if ((st = pg_sms(&sms))) return st;
    const uint32_t lanes = 128 / (hd >> 4), all = heads + 2 * kv->kv_heads, most = (all + lanes - 1) / lanes;
    uint32_t gy = (uint32_t)((8ull * sms + tokens - 1) / tokens);
    if (gy > most) gy = most;
    if (gy < 1) gy = 1;
    const dim3 grid((uint32_t)tokens, gy);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool bf = kv->dtype == QB200_BF16;
    cudaError_t e;
    if (x_dtype == QB200_F32) e = bf ? launch_append<float, __nv_bfloat16>(a, vec, grid, s) : launch_append<float, __half>(a, vec, grid, s);
    else if (x_dtype == QB200_BF16) e = bf ? launch_append<__nv_bfloat16, __nv_bfloat16>(a, vec, grid, s) : launch_append<__nv_bfloat16, __half>(a, vec, grid, s);
    else e = bf ? launch_append<__half, __nv_bfloat16>(a, vec, grid, s) : launch_append<__half, __half>(a, vec, grid, s);
    QB_CUDA_TRY(e);
    return QB200_OK;
}

uint64_t qb200_paged_attention_scratch_floats(const qb200_paged_kv* kv, const qb200_paged_batch* batch, uint64_t tokens, uint32_t heads) {
    const char* who = "qb200_paged_attention_scratch_floats";
    uint32_t sms = 0;
    if (pg_check_cache(who, kv, batch, tokens) || pg_check_heads(who, kv, tokens, heads) || pg_sms(&sms)) return 0;
    return pg_plan(pg_args(kv, batch, tokens, heads), kv->head_dim, sms).floats;
}

qb200_status qb200_paged_attention(const qb200_paged_kv* kv, const qb200_paged_batch* batch, const void* q, uint64_t q_stride, uint64_t tokens,
                                   uint32_t heads, float scale, float softcap, const float* slopes, const int32_t* prefix_lens, int32_t causal,
                                   float* scratch, void* out, float* lse, void* stream) {
    qb200_status st = pg_check_attention("qb200_paged_attention", kv, batch, q, q_stride, tokens, heads, scale, softcap, scratch, out);
    if (st) return st;
    if (tokens == 0) return QB200_OK;
    uint32_t sms = 0;
    if ((st = pg_sms(&sms))) return st;
    PgArgs a = pg_args(kv, batch, tokens, heads);
    a.q = q;
    a.q_stride = q_stride;
    a.prefix_lens = prefix_lens;
    a.causal = causal ? 1 : 0;
    a.out = static_cast<uint16_t*>(out);
    a.lse = lse;
    pg_scores(a, scale, softcap, slopes);
    return pg_phase("qb200_paged_attention", a, kv->dtype, kv->head_dim, sms, scratch, static_cast<cudaStream_t>(stream));
}

// The prefix phase leaves the state (m, l, acc) of every row in 32 bits; the phase over the sequences' own keys joins it
// as it writes the row.  (Joining the ranges of the prefix there too, instead of in a kernel of their own, put 18
// dependent reads behind every unit: 95 us instead of 63 for 64 sequences behind 8192 keys.)
static PgArgs prefix_args(const PgArgs& own, const int32_t* pages, uint64_t prefix_len, uint32_t hd, float* rows) {
    PgArgs a = own;
    a.shared = (uint32_t)prefix_len;
    a.table = pages;
    a.causal = 0;
    a.width = (uint32_t)((prefix_len + (1u << a.ps_log) - 1) >> a.ps_log);
    a.rows_acc = rows;
    a.rows_ml = rows + (uint64_t)a.tokens * a.group * a.kv_heads * hd;
    return a;
}
static uint64_t prefix_rows_floats(const PgArgs& a, uint32_t hd) { return ((uint64_t)a.tokens * a.group * a.kv_heads * (hd + 2) + 3) / 4 * 4; }

uint64_t qb200_shared_prefix_scratch_floats(const qb200_paged_kv* kv, const qb200_paged_batch* batch, uint64_t prefix_len, uint64_t tokens,
                                            uint32_t heads) {
    const char* who = "qb200_shared_prefix_scratch_floats";
    uint32_t sms = 0;
    if (pg_check_cache(who, kv, batch, tokens) || pg_check_heads(who, kv, tokens, heads) || pg_check_prefix(who, kv, batch, prefix_len) || pg_sms(&sms)) return 0;
    const PgArgs own = pg_args(kv, batch, tokens, heads);
    const uint64_t x = pg_plan(own, kv->head_dim, sms).floats;
    const uint64_t y = pg_plan(prefix_args(own, nullptr, prefix_len, kv->head_dim, nullptr), kv->head_dim, sms).floats;
    return prefix_rows_floats(own, kv->head_dim) + (x > y ? x : y);  // the phases follow one another: one area for both
}

qb200_status qb200_shared_prefix_attention(const qb200_paged_kv* kv, const qb200_paged_batch* batch, const int32_t* prefix_pages,
                                           uint64_t prefix_len, const void* q, uint64_t q_stride, uint64_t tokens, uint32_t heads, float scale,
                                           float softcap, const float* slopes, float* scratch, void* out, float* lse, void* stream) {
    const char* who = "qb200_shared_prefix_attention";
    qb200_status st = pg_check_attention(who, kv, batch, q, q_stride, tokens, heads, scale, softcap, scratch, out);
    if (st) return st;
    if (!prefix_pages) return fail(QB200_ERR_INVALID_PARAM, std::string(who) + ": no prefix (call qb200_paged_attention)");
    if ((st = pg_check_prefix(who, kv, batch, prefix_len))) return st;
    if (tokens == 0) return QB200_OK;
    uint32_t sms = 0;
    if ((st = pg_sms(&sms))) return st;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    PgArgs a = pg_args(kv, batch, tokens, heads);
    a.q = q;
    a.q_stride = q_stride;
    pg_scores(a, scale, softcap, slopes);
    if (!scratch) return fail(QB200_ERR_INVALID_PARAM, std::string(who) + ": the call needs its scratch");
    float* phase = scratch + prefix_rows_floats(a, kv->head_dim);
    const PgArgs p = prefix_args(a, prefix_pages, prefix_len, kv->head_dim, scratch);
    if ((st = pg_phase(who, p, kv->dtype, kv->head_dim, sms, phase, s))) return st;
    a.base_acc = p.rows_acc;
    a.base_ml = p.rows_ml;
    a.out = static_cast<uint16_t*>(out);
    a.lse = lse;
    return pg_phase(who, a, kv->dtype, kv->head_dim, sms, phase, s);
}

qb200_status qb200_paged_set_spin_limit(uint32_t polls) {
    if (polls == 0) return fail(QB200_ERR_INVALID_PARAM, "qb200_paged_set_spin_limit: the limit must be positive");
    g_pg_spin_limit.store(polls, std::memory_order_relaxed);
    return QB200_OK;
}

qb200_status qb200_paged_check(const qb200_paged_kv* kv, void* stream) {
    if (!kv || !kv->status_dev) return fail(QB200_ERR_INVALID_PARAM, "qb200_paged_check: null cache");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int32_t word = 0;
    QB_CUDA_TRY(cudaMemcpyAsync(&word, kv->status_dev, sizeof(word), cudaMemcpyDeviceToHost, s));
    QB_CUDA_TRY(cudaStreamSynchronize(s));
    if (word == 0) return QB200_OK;
    QB_CUDA_TRY(cudaMemsetAsync(kv->status_dev, 0, sizeof(word), s));
    if (word == QB200_ERR_LENGTH)
        return fail(QB200_ERR_LENGTH, "paged cache: a length did not fit its call (more keys than the table holds, a negative length, or cu_q out of order)");
    if (word == QB200_ERR_INVALID_PARAM)
        return fail(QB200_ERR_INVALID_PARAM, "paged cache: a page number outside the pool, or a position outside the table of angles");
    return fail((qb200_status)word, "paged cache: a kernel's wait ran out");
}

}  // extern "C"
