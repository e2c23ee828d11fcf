// Paged attention for few rows per K/V head (single tokens, drafts): bounded by the bytes of K and V (64 sequences of 1 to
// 8192 keys, 32 / 8 heads of 128: 160 us, 6.7 TB/s; 16 of 1024 keys, 32 / 32 heads: 43 us, 6.3 TB/s).
//
// A unit is (sequence of at most 16 packed rows, K/V head); it has ceil(keys / 64) tiles of 64 keys.  The tiles of all
// units, end to end, are cut into equal runs, one per CTA, so that ragged batches and one long sequence keep every SM
// equally busy; a unit cut by a run's end leaves partial results (m, l, acc) that a second kernel joins.  The lengths
// are read on the device, so a captured call follows them.
//
// A CTA has four warps and each takes 16 of a tile's keys on its own: its K and V rows travel by 16-byte asynchronous
// copies through a ring of its own (no barrier in the loop), S = Q K^T and O += P V run on the tensor pipe
// (m16n8k16; the packed rows are the 16) and the softmax is one pass with a running maximum.  The ring runs on across
// units: while one unit's warps are joined and its rows written, the next one's keys are already under way.
// P enters the second product as the sum of two numbers of the cache's type (an error of half a step of half a step, 2^-16 in
// bf16): rounded once, its error would reach that of the output's own rounding, and the tensor pipe has the room.  Where a
// call has at most 8 rows a unit, the second parts take the places of rows 8 .. 15 of the same instruction and the two
// results are added at the unit's end (16 sequences of 1024 keys: 42.7 us against 43.6 by a second product, 43.2 with P rounded
// once; 64 of 1 to 8192 keys: 159.6, 161.1 and 160.2; capped 160.5, 164.1 and 162.5).
#include <string>

#include "paged.cuh"

namespace qb {

constexpr uint32_t PR_WARPS = 4, PR_KEYS = 16, PR_TILE = PR_WARPS * PR_KEYS, PR_ROWS = PG_FEW_ROWS;
static_assert(PR_ROWS == 16, "the rows of one tensor instruction");
template <uint32_t HD> struct PrShape {
    static constexpr uint32_t ROW = HD * 2, STAGE = 2 * PR_KEYS * ROW;  // bytes of a row; of a stage (K, then V)
    static constexpr uint32_t STAGES = HD == 128 ? 3 : 6, WARP = STAGES * STAGE, RING = PR_WARPS * WARP;
    static constexpr uint32_t PASS = 4, ACC = HD + 4;  // rows that the warps join at a time, floats between them (no bank conflicts)
    static constexpr uint32_t JOIN = RING, ML = JOIN + PR_WARPS * PASS * ACC * 4, Q = ML + PR_WARPS * 2 * PR_ROWS * 4;
    static constexpr uint32_t SMEM = Q + PR_ROWS * ROW;
    static constexpr uint32_t PART = PR_ROWS * (HD + 2);  // floats of one partial result: m, l [16] each, acc [16][hd]
    static_assert(2 * (SMEM + 4096) <= 228 * 1024, "two CTAs per SM");
};

__device__ __forceinline__ uint32_t pr_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes to shared memory; `bytes` = 0 writes zeros and reads nothing.  Keys and values are read once a step, with other
// layers' in between: first to leave the L2 (16 sequences of 1024 keys: 46.7 us against 48.4, one of 131072: 86.6 against 88.6).
__device__ __forceinline__ uint64_t pr_once() {
    uint64_t policy;
    asm("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(policy));
    return policy;
}
__device__ __forceinline__ void pr_copy16(uint32_t dst, const void* src, uint32_t bytes, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(policy) : "memory");
}
__device__ __forceinline__ void pr_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void pr_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void pr_ldsm(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pr_ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pr_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pr_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Tiles of one unit of a sequence (a unit without keys still has one: it writes zeros), and of all its units; none
// where the sequence has more rows than a unit holds (the prompt kernel takes those) or none.  The host has made sure
// that all tiles of a call are fewer than 2^32.
__device__ __forceinline__ uint32_t pr_tiles(const PgSeq& s) { return max(1u, (s.kv + PR_TILE - 1) / PR_TILE); }
__device__ __forceinline__ uint32_t pr_weight(const PgArgs& a, const PgSeq& s) {
    const uint64_t rows = (uint64_t)s.q_len * a.group;
    return rows == 0 || rows > PG_FEW_ROWS ? 0 : a.kv_heads * pr_tiles(s);
}

// Tiles of a CTA up to which units are given to clusters (where the CTAs leave SMs idle, and where they do not).  Clusters
// need no search and no second launch, equal runs balance long ragged batches and cut single long sequences finer.  Us
// by clusters / by runs, K/V heads x sequences x keys: 8 x 1 x 1024 5.1 / 7.1, 8 x 1 x 4096 8.8 / 10.6, 8 x 1 x 16384 25 / 19;
// 32 x 16 x 1024 42 / 46, 8 x 64 x 2048 80 / 84 (lengths up to 2048: 51 / 54), 8 x 64 x 8192 301 / 313 (up to 8192: 190 / 172).
constexpr uint32_t PR_SHORT = 8, PR_LONG = 32;
// Steps (16 rows against 64 keys of a K/V head) up to which a call of several row tiles stays here, us here / by the prompt
// kernel: 8 K/V heads, 512 rows, 128 keys 6.6 / 10.4; 128 rows, 1000 keys 9.5 / 15.2; 64 tokens of 4 heads behind 1000
// shared keys (2048 steps) 19.8 / 22.4, behind 4000 (8064 steps) 39 / 28.
constexpr uint64_t PR_STEPS = 6144;

// Sequences whose lengths the CTA keeps in shared memory: the first ones of the call.
constexpr uint32_t PR_KEPT = PR_WARPS * 32;

// The CTA's run of tiles, [run0, run1) of the total, and the sequence that holds tile run0 (first: its first tile).
// Runs differ by at most one tile, the longer ones first.
struct PrRun {
    PgSeq s;
    uint32_t run0, run1, first, seq;
    uint32_t base, extra;  // tiles of the shorter runs, how many runs are one longer
};
// All threads of the CTA take part; false where it has no run (the same for all).  Long batches' lengths are read twice, for the total
// and to find the run: what is found is kept as it was found, and where another stream's writes in between leave nothing to find
// there is no run.
__device__ __forceinline__ bool pr_find_run(const PgArgs& a, uint32_t seqs, PgSeq* kept, PrRun& r) {
    __shared__ uint32_t s_warp[PR_WARPS], s_first, s_seq;
    __shared__ PgSeq s_found;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    PgSeq mine = {};
    uint32_t sum = 0, w0 = 0;
    for (uint32_t b = tid; b < seqs; b += PR_KEPT) {
        const PgSeq s = pg_seq(a, b);
        const uint32_t w = pr_weight(a, s);
        if (b < PR_KEPT) {
            mine = s;
            w0 = w;
        }
        sum += w;
    }
    kept[tid] = mine;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) s_warp[warp] = sum;
    if (tid == 0) s_seq = 0xFFFFFFFFu;
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < PR_WARPS; w++) total += s_warp[w];
    const uint32_t ctas = min(gridDim.x, total), i = blockIdx.x;
    if (i >= ctas) return false;
    r.base = total / ctas;
    r.extra = total - r.base * ctas;
    r.run0 = i * r.base + min(i, r.extra);
    r.run1 = r.run0 + r.base + (i < r.extra ? 1 : 0);
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < seqs; b0 += PR_KEPT) {
        const uint32_t b = b0 + tid;
        uint32_t w = w0;
        if (b0) {
            w = 0;
            if (b < seqs) {
                mine = pg_seq(a, b);
                w = pr_weight(a, mine);
            }
        }
        uint32_t incl = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xFFFFFFFFu, incl, o);
            if (lane >= (uint32_t)o) incl += t;
        }
        __syncthreads();  // s_warp is read by all before it is written again
        if (lane == 31) s_warp[warp] = incl;
        __syncthreads();
        uint32_t excl = before + incl - w;
#pragma unroll
        for (uint32_t k = 0; k < PR_WARPS; k++) {
            if (k < warp) excl += s_warp[k];
            before += s_warp[k];
        }
        if (excl <= r.run0 && r.run0 - excl < w) {
            s_seq = b;
            s_first = excl;
            s_found = mine;
        }
        __syncthreads();
        if (s_seq != 0xFFFFFFFFu) break;
    }
    if (s_seq == 0xFFFFFFFFu) {
        if (tid == 0) pg_report(a.status, QB200_ERR_LENGTH);
        return false;
    }
    r.s = s_found;
    r.seq = s_seq;
    r.first = s_first;
    return true;
}

// A place in the CTA's run: tile t of K/V head kvh of sequence b.
struct PrAt {
    PgSeq s;
    uint32_t b, kvh, t, tiles, left;  // left: tiles of the run from here on
};
__device__ __forceinline__ PgSeq pr_seq(const PgArgs& a, const PgSeq* kept, uint32_t b) { return b < PR_KEPT ? kept[b] : pg_seq(a, b); }
// n tiles further (not past the unit's end).
__device__ __forceinline__ void pr_advance(const PgArgs& a, const PgSeq* kept, uint32_t seqs, PrAt& p, uint32_t n) {
    p.left -= n;
    p.t += n;
    if (p.left == 0 || p.t < p.tiles) return;
    p.t = 0;
    if (++p.kvh < a.kv_heads) return;
    p.kvh = 0;
    do {  // the run goes on, so there is one (but for lengths that another stream changes meanwhile)
        if (++p.b >= seqs) {
            p.left = 0;
            return;
        }
        p.s = pr_seq(a, kept, p.b);
    } while (pr_weight(a, p.s) == 0);
    p.tiles = pr_tiles(p.s);
}

// What a warp holds of a unit: a thread has rows lane / 4 and lane / 4 + 8.
template <uint32_t HD> struct PrState {
    float m[2], l[2], o[HD / 8][4];
    uint32_t lim[2];  // keys the rows see, and the bias they get
    float slope[2];
    int32_t pos[2];
};
template <uint32_t HD, bool SCORED>
__device__ __forceinline__ void pr_begin(const PgArgs& a, const PgSeq& sq, uint32_t kvh, uint32_t row0, PrState<HD>& u) {
#pragma unroll
    for (uint32_t i = 0; i < 2; i++) {
        const uint32_t r = row0 + ((threadIdx.x & 31) >> 2) + 8 * i;
        u.m[i] = -INFINITY;
        u.l[i] = 0.0f;
        u.lim[i] = 0;
        u.slope[i] = 0.0f;
        u.pos[i] = 0;
        if (r < sq.q_len * a.group) {
            u.lim[i] = pg_limit(sq, r / a.group);
            if (SCORED && a.slopes) {
                u.slope[i] = a.slopes[kvh * a.group + r % a.group] * PG_LOG2E;
                u.pos[i] = pg_position(a, sq, r / a.group);
            }
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < HD / 8; k++) u.o[k][0] = u.o[k][1] = u.o[k][2] = u.o[k][3] = 0.0f;
}
// A 16-byte chunk of the unit's 16 rows of Q, from row0 on (zeros past the last row).
template <uint32_t HD>
__device__ __forceinline__ uint4 pr_load_q(const PgArgs& a, const PgSeq& sq, uint32_t kvh, uint32_t row0, uint32_t id) {
    const uint32_t r = row0 + id / (HD / 8), c = id % (HD / 8);
    if (r >= sq.q_len * a.group) return make_uint4(0, 0, 0, 0);
    return *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + (uint64_t)(sq.q0 + r / a.group) * a.q_stride +
                                           (uint64_t)(kvh * a.group + r % a.group) * HD + c * 8);
}
template <uint32_t HD> __device__ __forceinline__ uint32_t pr_q_place(uint32_t id) {
    const uint32_t r = id / (HD / 8), c = id % (HD / 8);
    return r * (HD * 2) + ((c ^ (r & 7)) << 4);
}
template <uint32_t HD> __device__ __forceinline__ void pr_q_fragments(uint32_t q_s, uint32_t (&qf)[HD / 16][4]) {
    const uint32_t lane = threadIdx.x & 31, r = (((lane >> 3) & 1) << 3) | (lane & 7), sub = lane >> 4;
#pragma unroll
    for (uint32_t ks = 0; ks < HD / 16; ks++) pr_ldsm(q_s + r * (HD * 2) + (((ks * 2 + sub) ^ (r & 7)) << 4), qf[ks]);
}
// 16 keys of a page and head to a stage (K, then V; 16-byte chunk c of a row at c ^ (row & 7)): `valid` of them, the
// others are zeros, whatever the page holds there, and so are all keys of a page that is not in the pool.
template <uint32_t HD>
__device__ __forceinline__ void pr_copy_keys(const PgArgs& a, uint32_t dst, int32_t page, uint32_t kvh, uint32_t key, uint32_t valid, uint64_t once) {
    constexpr uint32_t CH = HD / 8, ROW = HD * 2;
    if (valid && (uint32_t)page >= a.n_pages) {
        pg_report(a.status, QB200_ERR_INVALID_PARAM);
        valid = 0;
    }
    const uint64_t base = valid ? (((uint64_t)(uint32_t)page * a.kv_heads + kvh) << a.ps_log) + (key & ((1u << a.ps_log) - 1)) : 0;
#pragma unroll
    for (uint32_t i = 0; i < PR_KEYS * CH / 32; i++) {
        const uint32_t id = i * 32 + (threadIdx.x & 31), row = id / CH, c = id % CH, bytes = row < valid ? 16u : 0u;
        const uint64_t src = (base + (bytes ? row : 0)) * HD + c * 8;
        const uint32_t d = dst + row * ROW + ((c ^ (row & 7)) << 4);
        pr_copy16(d, a.k + src, bytes, once);
        pr_copy16(d + PR_KEYS * ROW, a.v + src, bytes, once);
    }
}
// One tile: the warp's 16 keys, from `first` on, in the stage at ks_s.  LIGHT: no unit of the call has more than 8 rows, and
// the second parts of their weights take the places of rows 8 .. 15.
template <typename T, uint32_t HD, bool SCORED, bool LIGHT>
__device__ __forceinline__ void pr_step(const PgArgs& a, uint32_t ks_s, uint32_t first, const uint32_t (&qf)[HD / 16][4], PrState<HD>& u) {
    using S = PrShape<HD>;
    constexpr uint32_t KS = HD / 16, NP = HD / 16;
    const uint32_t lane = threadIdx.x & 31, part4 = lane & 3, vs_s = ks_s + PR_KEYS * S::ROW;
    float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
    {
        const uint32_t key = ((lane >> 4) << 3) | (lane & 7), sub = (lane >> 3) & 1;
#pragma unroll
        for (uint32_t ks = 0; ks < KS; ks++) {
            uint32_t kf[4];
            pr_ldsm(ks_s + key * S::ROW + (((ks * 2 + sub) ^ (key & 7)) << 4), kf);
            pr_mma(s[0], qf[ks], kf[0], kf[1], T());
            pr_mma(s[1], qf[ks], kf[2], kf[3], T());
        }
    }
    const uint32_t key0 = first + part4 * 2;
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (uint32_t k = 0; k < 2; k++)
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t r = i >> 1, key = key0 + k * 8 + (i & 1);
            if (LIGHT && r) continue;
            float x = s[k][i] * a.score_mul;
            if (SCORED) {
                if (a.cap_mul != 0.0f) x = pg_cap(x, a.cap_mul);
                x = fmaf(-u.slope[r], fabsf((float)(u.pos[r] - (int32_t)key)), x);
            }
            x = key < u.lim[r] ? x : -INFINITY;
            s[k][i] = x;
            mx[r] = fmaxf(mx[r], x);
        }
    float f[2], ms[2];
#pragma unroll
    for (uint32_t r = 0; r < 2; r++) {
        if (LIGHT && r) {
            f[1] = f[0];
            break;
        }
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xFFFFFFFFu, mx[r], 1));
        mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xFFFFFFFFu, mx[r], 2));
        const float mn = fmaxf(u.m[r], mx[r]);
        ms[r] = mn == -INFINITY ? 0.0f : mn;
        f[r] = mn == -INFINITY ? 1.0f : pg_exp2(u.m[r] - mn);  // (a row without keys so far has nothing to scale)
        u.m[r] = mn;
        u.l[r] *= f[r];
    }
    if (__any_sync(0xFFFFFFFFu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
        for (uint32_t k = 0; k < 2 * NP; k++) {
            u.o[k][0] *= f[0];
            u.o[k][1] *= f[0];
            u.o[k][2] *= f[1];
            u.o[k][3] *= f[1];
        }
    }
    uint32_t pf[4], pl[4];
#pragma unroll
    for (uint32_t k = 0; k < 2; k++)
#pragma unroll
        for (uint32_t r = 0; r < (LIGHT ? 1 : 2); r++) {
            const float p0 = pg_exp2(s[k][2 * r] - ms[r]), p1 = pg_exp2(s[k][2 * r + 1] - ms[r]);
            u.l[r] += p0 + p1;
            pf[k * 2 + r] = PgType<T>::pack(p0, p1);
            const float2 h = PgType<T>::widen2(pf[k * 2 + r]);
            pl[k * 2 + r] = PgType<T>::pack(p0 - h.x, p1 - h.y);
            if (LIGHT) pf[k * 2 + 1] = pl[k * 2];
        }
    {
        const uint32_t key = (((lane >> 3) & 1) << 3) | (lane & 7), sub = lane >> 4;
#pragma unroll
        for (uint32_t k = 0; k < NP; k++) {
            uint32_t vf[4];
            pr_ldsm_t(vs_s + key * S::ROW + (((k * 2 + sub) ^ (key & 7)) << 4), vf);
            pr_mma(u.o[2 * k], pf, vf[0], vf[1], T());
            pr_mma(u.o[2 * k + 1], pf, vf[2], vf[3], T());
            if (!LIGHT) {
                pr_mma(u.o[2 * k], pl, vf[0], vf[1], T());
                pr_mma(u.o[2 * k + 1], pl, vf[2], vf[3], T());
            }
        }
    }
}
// The sums of a thread's two rows over the four threads that share them, and the row's (m, l) to ml [2][16].
template <uint32_t HD, bool LIGHT> __device__ __forceinline__ void pr_end(PrState<HD>& u, float* ml) {
    const uint32_t lane = threadIdx.x & 31, quad = lane >> 2;
    if (LIGHT) {
#pragma unroll
        for (uint32_t k = 0; k < HD / 8; k++) {
            u.o[k][0] += u.o[k][2];
            u.o[k][1] += u.o[k][3];
        }
    }
#pragma unroll
    for (uint32_t r = 0; r < 2; r++) {
        u.l[r] += __shfl_xor_sync(0xFFFFFFFFu, u.l[r], 1);
        u.l[r] += __shfl_xor_sync(0xFFFFFFFFu, u.l[r], 2);
    }
    if ((lane & 3) == 0) {
        ml[quad] = u.m[0];
        ml[quad + 8] = u.m[1];
        ml[PR_ROWS + quad] = u.l[0];
        ml[PR_ROWS + quad + 8] = u.l[1];
    }
}
// Rows [p0, p0 + PASS) of the warp's accumulator to the join area.
template <uint32_t HD> __device__ __forceinline__ void pr_put_rows(const PrState<HD>& u, float* j_acc, uint32_t p0) {
    using S = PrShape<HD>;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (uint32_t i = 0; i < 2; i++) {
        const uint32_t r = (lane >> 2) + 8 * i - p0;
        if (r < S::PASS) {
            float* to = j_acc + (warp * S::PASS + r) * S::ACC + (lane & 3) * 2;
#pragma unroll
            for (uint32_t k = 0; k < HD / 8; k++) *reinterpret_cast<float2*>(to + k * 8) = make_float2(u.o[k][2 * i], u.o[k][2 * i + 1]);
        }
    }
}
// Four columns of row r over the CTA's warps.
template <uint32_t HD>
__device__ __forceinline__ float4 pr_join_warps(const float* j_acc, const float* j_ml, uint32_t r, uint32_t p0, uint32_t col, float& M, float& L) {
    using S = PrShape<HD>;
    M = -INFINITY;
#pragma unroll
    for (uint32_t w = 0; w < PR_WARPS; w++) M = fmaxf(M, j_ml[w * 2 * PR_ROWS + r]);
    L = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (uint32_t w = 0; w < PR_WARPS; w++) {
        const float g = pg_weight(j_ml[w * 2 * PR_ROWS + r], M);
        const float4 e = *reinterpret_cast<const float4*>(j_acc + (w * S::PASS + r - p0) * S::ACC + col);
        L = fmaf(j_ml[w * 2 * PR_ROWS + PR_ROWS + r], g, L);
        v.x = fmaf(e.x, g, v.x);
        v.y = fmaf(e.y, g, v.y);
        v.z = fmaf(e.z, g, v.z);
        v.w = fmaf(e.w, g, v.w);
    }
    return v;
}

template <typename T, uint32_t HD, bool SCORED, bool LIGHT>
__global__ void __launch_bounds__(PR_WARPS * 32, 2) k_paged_rows(const __grid_constant__ PgArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    using S = PrShape<HD>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ PgSeq kept[PR_KEPT];
    const uint32_t tid = threadIdx.x, warp = tid >> 5;
    int32_t* meta = a.meta + blockIdx.x * 8;
    if (tid == 0) meta[0] = -1;
    PrRun run;
    const uint32_t seqs = a.shared ? 1 : a.batch;
    if (!pr_find_run(a, seqs, kept, run)) return;
    const uint32_t ring_s = pr_smem(smem + warp * S::WARP), q_s = pr_smem(smem + S::Q);
    float* j_acc = reinterpret_cast<float*>(smem + S::JOIN);
    float* j_ml = reinterpret_cast<float*>(smem + S::ML);

    PrAt here, ahead;  // what is computed and what is fetched
    here.b = run.seq;
    here.s = run.s;
    here.tiles = pr_tiles(here.s);
    here.kvh = (run.run0 - run.first) / here.tiles;
    here.t = run.run0 - run.first - here.kvh * here.tiles;
    here.left = run.run1 - run.run0;
    ahead = here;

    // ---- the ring: the warp's 16 keys of one tile a stage.  The next tile's page number is read a step before it is needed. ----
    const uint64_t once = pr_once();
    int32_t n_page = 0;
    uint32_t n_kvh = 0, n_key = 0, n_valid = 0;
    bool n_there = false;
    auto look = [&]() {
        n_there = ahead.left != 0;
        if (!n_there) return;
        n_key = ahead.t * PR_TILE + warp * PR_KEYS;
        n_valid = n_key < ahead.s.kv ? min(ahead.s.kv - n_key, PR_KEYS) : 0;
        n_kvh = ahead.kvh;
        if (n_valid) n_page = a.table[(a.shared ? 0 : (uint64_t)ahead.b * a.table_stride) + (n_key >> a.ps_log)];
        pr_advance(a, kept, seqs, ahead, 1);
    };
    auto fetch = [&](uint32_t st) {
        if (n_there) {
            pr_copy_keys<HD>(a, ring_s + st * S::STAGE, n_page, n_kvh, n_key, n_valid, once);
            look();
        }
        pr_commit();
    };

    // ---- Q of a unit: loaded while the unit before it is joined, then through shared memory into fragments ----
    constexpr uint32_t QN = PR_ROWS * (HD / 8) / 128;  // 16-byte chunks a thread brings
    uint4 q_in[QN];
    auto bring_q = [&](const PrAt& p) {
#pragma unroll
        for (uint32_t i = 0; i < QN; i++) q_in[i] = pr_load_q<HD>(a, p.s, p.kvh, 0, i * 128 + tid);
    };

    bring_q(here);
    look();
#pragma unroll
    for (uint32_t i = 0; i + 1 < S::STAGES; i++) fetch(i);
    uint32_t st = 0, slot = 0;  // slot: the CTA's first unit, where it is a part, goes to its slot 0, the last one to slot 1
    while (true) {
        // ---- a unit ----
#pragma unroll
        for (uint32_t i = 0; i < QN; i++) *reinterpret_cast<uint4*>(smem + S::Q + pr_q_place<HD>(i * 128 + tid)) = q_in[i];
        __syncthreads();
        uint32_t qf[HD / 16][4];
        pr_q_fragments<HD>(q_s, qf);
        const PgSeq sq = here.s;
        const uint32_t kvh = here.kvh, rows = sq.q_len * a.group, t0 = here.t, n = min(here.tiles - t0, here.left);
        const bool whole = n == here.tiles;
        PrState<HD> u;
        pr_begin<HD, SCORED>(a, sq, kvh, 0, u);

        for (uint32_t t = t0; t < t0 + n; t++) {
            pr_wait<S::STAGES - 2>();
            __syncwarp();
            const uint32_t ks_s = ring_s + st * S::STAGE;
            pr_step<T, HD, SCORED, LIGHT>(a, ks_s, t * PR_TILE + warp * PR_KEYS, qf, u);
            __syncwarp();  // every lane is done with the stage that the next fetch overwrites: the one before this
            fetch(st == 0 ? S::STAGES - 1 : st - 1);
            if (++st == S::STAGES) st = 0;
        }

        // ---- its end: on to the next unit's Q, then the warps' states are joined, PASS rows at a time ----
        const uint32_t first_tile = run.run1 - here.left;
        pr_advance(a, kept, seqs, here, n);
        const bool more = here.left != 0;
        if (more) bring_q(here);
        pr_end<HD, LIGHT>(u, j_ml + warp * 2 * PR_ROWS);
        float* part = a.parts + ((uint64_t)blockIdx.x * 2 + slot) * S::PART;
        if (!whole && t0 == 0 && tid == 0) {  // a unit that starts here and goes on: what the second kernel joins
            const uint32_t x = first_tile + pr_tiles(sq) - 1, cut = run.extra * (run.base + 1);
            meta[1] = (int32_t)slot;
            meta[2] = (int32_t)sq.q0;
            meta[3] = (int32_t)rows;
            meta[4] = (int32_t)kvh;
            // the CTA that has its last tile (one of the grid's, whatever the lengths have become)
            meta[0] = (int32_t)min(x < cut ? x / (run.base + 1) : run.extra + (x - cut) / run.base, gridDim.x - 1);
        }
        constexpr uint32_t PER = HD / 4;  // threads of a row
        for (uint32_t p0 = 0; p0 < rows; p0 += S::PASS) {
            if (p0) __syncthreads();  // the rows before have been read
            pr_put_rows<HD>(u, j_acc, p0);
            __syncthreads();
#pragma unroll 1
            for (uint32_t r = p0 + tid / PER; r < min(rows, p0 + S::PASS); r += PR_WARPS * 32 / PER) {
                const uint32_t col = (tid % PER) * 4;
                float M, L;
                const float4 v = pr_join_warps<HD>(j_acc, j_ml, r, p0, col, M, L);
                if (whole) {
                    pg_emit<T, HD>(a, sq.q0 + r / a.group, kvh * a.group + r % a.group, col, M, L, v);
                } else {
                    if (col == 0) {
                        part[r] = M;
                        part[PR_ROWS + r] = L;
                    }
                    *reinterpret_cast<float4*>(part + 2 * PR_ROWS + r * HD + col) = v;
                }
            }
        }
        if (!more) break;
        slot = 1;
        __syncthreads();  // the join area is free again
    }
    pr_wait<0>();
}

// The same for tables of moderate length, in one launch and without a search: a unit has a cluster of 2^c_log CTAs, each
// takes an equal range of its tiles, and their states meet in the cluster's shared memory.  Where the call has few rows in
// all, sequences of up to row_tiles * 16 rows are taken, 16 rows a unit (side by side, so that they share the L2).
template <typename T, uint32_t HD, bool SCORED, bool LIGHT>
__global__ void __launch_bounds__(PR_WARPS * 32, 2) k_paged_units(const __grid_constant__ PgArgs a, uint32_t c_log, uint32_t row_tiles) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    using S = PrShape<HD>;
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t tid = threadIdx.x, warp = tid >> 5;
    const uint32_t rank = blockIdx.x & ((1u << c_log) - 1), unit = blockIdx.x >> c_log, b = unit / (a.kv_heads * row_tiles);
    const uint32_t in = unit - b * a.kv_heads * row_tiles, kvh = in / row_tiles, row0 = (in - kvh * row_tiles) * PR_ROWS;
    const PgSeq sq = pg_seq(a, b);
    const uint32_t all_rows = sq.q_len * a.group;
    if (all_rows <= row0 || all_rows > row_tiles * PR_ROWS) return;  // the whole cluster alike
    const uint32_t rows = min(PR_ROWS, all_rows - row0);
    const uint32_t keys = pg_limit(sq, (row0 + rows - 1) / a.group);  // that the unit's last token sees (the most)
    const uint32_t ring_s = pr_smem(smem + warp * S::WARP), q_s = pr_smem(smem + S::Q);
    float* j_acc = reinterpret_cast<float*>(smem + S::JOIN);
    float* j_ml = reinterpret_cast<float*>(smem + S::ML);
    const uint64_t once = pr_once();
    const uint32_t tiles = max(1u, (keys + PR_TILE - 1) / PR_TILE), t0 = tiles * rank >> c_log, t1 = tiles * (rank + 1) >> c_log;
    const int32_t* table = a.table + (a.shared ? 0 : (uint64_t)b * a.table_stride);
    uint32_t ahead = t0;  // the next tile to fetch, and its page
    int32_t page = 0;
    auto look = [&]() {
        const uint32_t key = ahead * PR_TILE + warp * PR_KEYS;
        if (ahead < t1 && key < keys) page = table[key >> a.ps_log];
    };
    auto fetch = [&](uint32_t st) {
        if (ahead < t1) {
            const uint32_t key = ahead * PR_TILE + warp * PR_KEYS;
            pr_copy_keys<HD>(a, ring_s + st * S::STAGE, page, kvh, key, key < keys ? min(keys - key, PR_KEYS) : 0, once);
            ahead++;
            look();
        }
        pr_commit();
    };
    constexpr uint32_t QN = PR_ROWS * (HD / 8) / 128;
    uint4 q_in[QN];
#pragma unroll
    for (uint32_t i = 0; i < QN; i++) q_in[i] = pr_load_q<HD>(a, sq, kvh, row0, i * 128 + tid);
    look();
#pragma unroll
    for (uint32_t i = 0; i + 1 < S::STAGES; i++) fetch(i);
#pragma unroll
    for (uint32_t i = 0; i < QN; i++) *reinterpret_cast<uint4*>(smem + S::Q + pr_q_place<HD>(i * 128 + tid)) = q_in[i];
    __syncthreads();
    uint32_t qf[HD / 16][4];
    pr_q_fragments<HD>(q_s, qf);
    PrState<HD> u;
    pr_begin<HD, SCORED>(a, sq, kvh, row0, u);
    uint32_t st = 0;
    for (uint32_t t = t0; t < t1; t++) {
        pr_wait<S::STAGES - 2>();
        __syncwarp();
        pr_step<T, HD, SCORED, LIGHT>(a, ring_s + st * S::STAGE, t * PR_TILE + warp * PR_KEYS, qf, u);
        __syncwarp();
        fetch(st == 0 ? S::STAGES - 1 : st - 1);
        if (++st == S::STAGES) st = 0;
    }
    pr_wait<0>();
    pr_end<HD, LIGHT>(u, j_ml + warp * 2 * PR_ROWS);
    // the CTA's state of its rows, in the ring's place (m, l and HD columns a row), then the cluster's
    constexpr uint32_t PER = HD / 4, ROW = HD + 4;
    float* mine = reinterpret_cast<float*>(smem);
    for (uint32_t p0 = 0; p0 < rows; p0 += S::PASS) {
        if (p0) __syncthreads();  // the rows before have been read
        pr_put_rows<HD>(u, j_acc, p0);
        __syncthreads();          // (the first one: no warp reads its ring any more)
#pragma unroll 1
        for (uint32_t r = p0 + tid / PER; r < min(rows, p0 + S::PASS); r += PR_WARPS * 32 / PER) {
            const uint32_t col = (tid % PER) * 4;
            float M, L;
            const float4 v = pr_join_warps<HD>(j_acc, j_ml, r, p0, col, M, L);
            if (c_log == 0) {
                pg_emit<T, HD>(a, sq.q0 + (row0 + r) / a.group, kvh * a.group + (row0 + r) % a.group, col, M, L, v);
                continue;
            }
            *reinterpret_cast<float4*>(mine + r * ROW + 4 + col) = v;
            if (col == 0) *reinterpret_cast<float2*>(mine + r * ROW) = make_float2(M, L);
        }
    }
    if (c_log == 0) return;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const uint32_t peers = 1u << c_log;
#pragma unroll 1
    for (uint32_t r = rank + (tid / PER << c_log); r < rows; r += (PR_WARPS * 32 / PER) << c_log) {
        const uint32_t col = (tid % PER) * 4, at = pr_smem(mine + r * ROW);
        float m[8], l[8];
        float4 e[8];
        float M = -INFINITY, L = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t p = 0; p < 8; p++) {
            m[p] = -INFINITY;
            l[p] = 0.0f;
            e[p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (p < peers) {
                uint32_t there;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(p));
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(m[p]), "=f"(l[p]) : "r"(there) : "memory");
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(e[p].x), "=f"(e[p].y), "=f"(e[p].z), "=f"(e[p].w) : "r"(there + 16 + col * 4) : "memory");
            }
        }
#pragma unroll
        for (uint32_t p = 0; p < 8; p++) M = fmaxf(M, m[p]);
#pragma unroll
        for (uint32_t p = 0; p < 8; p++) {
            const float g = pg_weight(m[p], M);
            L = fmaf(l[p], g, L);
            v.x = fmaf(e[p].x, g, v.x);
            v.y = fmaf(e[p].y, g, v.y);
            v.z = fmaf(e[p].z, g, v.z);
            v.w = fmaf(e[p].w, g, v.w);
        }
        pg_emit<T, HD>(a, sq.q0 + (row0 + r) / a.group, kvh * a.group + (row0 + r) % a.group, col, M, L, v);
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // no CTA leaves while its state is read
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Joins the partial results of the unit that starts in CTA blockIdx.x's run and ends in a later one's.  A block takes
// four of its rows, from 4 * blockIdx.y on; LANES groups of threads take every LANES-th part of a row (one sequence's
// keys may be cut into dozens: taken one after the other, 37 parts cost 18 us) and meet in shared memory.
template <typename T, uint32_t HD>
__global__ void __launch_bounds__(512) k_paged_rows_join(const __grid_constant__ PgArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    using S = PrShape<HD>;
    constexpr uint32_t PER = HD / 4, LANES = 512 / 4 / PER, U = 4;
    __shared__ float4 s_acc[4][LANES][PER];
    __shared__ float s_m[4][LANES], s_l[4][LANES];
    const int4 m0 = *reinterpret_cast<const int4*>(a.meta + blockIdx.x * 8);
    const uint32_t kvh = (uint32_t)a.meta[blockIdx.x * 8 + 4];
    if (m0.x < 0) return;
    const uint32_t last = (uint32_t)m0.x, slot0 = (uint32_t)m0.y, q0 = (uint32_t)m0.z, rows = (uint32_t)m0.w;
    const uint32_t piece = threadIdx.x % PER, col = piece * 4, k = threadIdx.x / PER % 4, lane = threadIdx.x / (4 * PER), r = blockIdx.y * 4 + k;
    if (blockIdx.y * 4 >= rows) return;
    float M = -INFINITY, L = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (r < rows) {
#pragma unroll 1
        for (uint32_t c0 = blockIdx.x + lane; c0 <= last; c0 += LANES * U) {
            float m[U], l[U];
            float4 e[U];
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                const uint32_t c = min(c0 + u * LANES, last);
                const float* p = a.parts + ((uint64_t)c * 2 + (c == blockIdx.x ? slot0 : 0)) * S::PART;
                m[u] = p[r];
                l[u] = p[PR_ROWS + r];
                e[u] = *reinterpret_cast<const float4*>(p + 2 * PR_ROWS + r * HD + col);
            }
            float Mn = M;
#pragma unroll
            for (uint32_t u = 0; u < U; u++)
                if (c0 + u * LANES <= last) Mn = fmaxf(Mn, m[u]);
            const float f = pg_weight(M, Mn);
            M = Mn;
            L *= f;
            v.x *= f;
            v.y *= f;
            v.z *= f;
            v.w *= f;
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                if (c0 + u * LANES > last) continue;
                const float g = pg_weight(m[u], M);
                L = fmaf(l[u], g, L);
                v.x = fmaf(e[u].x, g, v.x);
                v.y = fmaf(e[u].y, g, v.y);
                v.z = fmaf(e[u].z, g, v.z);
                v.w = fmaf(e[u].w, g, v.w);
            }
        }
        s_acc[k][lane][piece] = v;
        if (piece == 0) {
            s_m[k][lane] = M;
            s_l[k][lane] = L;
        }
    }
    __syncthreads();
    if (lane || r >= rows) return;
    M = s_m[k][0];
#pragma unroll
    for (uint32_t i = 1; i < LANES; i++) M = fmaxf(M, s_m[k][i]);
    const float f = pg_weight(s_m[k][0], M);
    L *= f;
    v.x *= f;
    v.y *= f;
    v.z *= f;
    v.w *= f;
#pragma unroll
    for (uint32_t i = 1; i < LANES; i++) {
        const float g = pg_weight(s_m[k][i], M);
        const float4 e = s_acc[k][i][piece];
        L = fmaf(s_l[k][i], g, L);
        v.x = fmaf(e.x, g, v.x);
        v.y = fmaf(e.y, g, v.y);
        v.z = fmaf(e.z, g, v.z);
        v.w = fmaf(e.w, g, v.w);
    }
    pg_emit<T, HD>(a, q0 + r / a.group, kvh * a.group + r % a.group, col, M, L, v);
}

// ---- host side ---------------------------------------------------------------------------------------------------

uint64_t pg_rows_most_tiles(const PgArgs& a) {
    const uint64_t keys = a.shared ? a.shared : (uint64_t)a.width << a.ps_log;
    return (a.shared ? 1 : (uint64_t)a.batch) * a.kv_heads * div_ceil(keys, PR_TILE);
}

PgRows pg_rows_plan(const PgArgs& a, uint32_t hd, uint32_t sms, uint32_t row_tiles) {
    PgRows how = {};
    how.row_tiles = row_tiles;
    const uint64_t most = pg_rows_most_tiles(a), seqs = (a.shared ? 1 : (uint64_t)a.batch) * a.kv_heads, units = seqs * row_tiles, tiles = most / seqs;
    // A cluster per unit, of up to 8 CTAs while all of them fit the SMs at once, where a CTA then has at most PR_SHORT
    // tiles, or at most PR_LONG and there are as many CTAs as SMs; equal runs otherwise.
    uint32_t c_log = 0;
    while (c_log < 3 && (units << (c_log + 1)) <= 2 * sms && (2u << c_log) <= tiles) c_log++;
    if (row_tiles > 1 && most * row_tiles > PR_STEPS) return how;
    if (units <= 0x7FFFFFFFull >> c_log && (tiles <= (uint64_t)PR_SHORT << c_log || (tiles <= (uint64_t)PR_LONG << c_log && units << c_log >= sms))) {
        how.units = true;
        how.c_log = c_log;
        how.grid = (uint32_t)(units << c_log);
        return how;
    }
    if (row_tiles > 1) return how;  // the equal runs take one tile of rows
    how.grid = (uint32_t)(most < 2 * sms ? most : 2 * sms);  // two CTAs per SM, fewer where the call cannot have as many tiles
    how.floats = (uint64_t)how.grid * 2 * PR_ROWS * (hd + 2) + (uint64_t)how.grid * 8;
    return how;
}

template <typename T, uint32_t HD, bool SCORED, bool LIGHT>
static qb200_status launch_rows(const PgArgs& a, const PgRows& how, cudaStream_t st) {
    static bool attr_set[64] = {};
    int dev = 0;
    QB_CUDA_TRY(cudaGetDevice(&dev));
    if (!attr_set[dev & 63]) {
        QB_CUDA_TRY(cudaFuncSetAttribute(k_paged_rows<T, HD, SCORED, LIGHT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PrShape<HD>::SMEM));
        QB_CUDA_TRY(cudaFuncSetAttribute(k_paged_units<T, HD, SCORED, LIGHT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PrShape<HD>::SMEM));
        attr_set[dev & 63] = true;
    }
    const uint32_t grid = how.grid;
    if (how.units) {
        QB_CUDA_TRY(pg_launch_cluster(k_paged_units<T, HD, SCORED, LIGHT>, dim3(grid), dim3(PR_WARPS * 32), PrShape<HD>::SMEM, st, 1u << how.c_log, a, how.c_log, how.row_tiles));
        return QB200_OK;
    }
    QB_CUDA_TRY(pg_launch(k_paged_rows<T, HD, SCORED, LIGHT>, dim3(grid), dim3(PR_WARPS * 32), PrShape<HD>::SMEM, st, a));
    const uint64_t rows = a.cu_q || a.shared ? (uint64_t)a.tokens * a.group : a.group;
    QB_CUDA_TRY(pg_launch(k_paged_rows_join<T, HD>, dim3(grid, (uint32_t)((rows < PR_ROWS ? rows : PR_ROWS) + 3) / 4), dim3(512), 0, st, a));
    return QB200_OK;
}

template <typename T, uint32_t HD>
static qb200_status launch_rows(const PgArgs& a, const PgRows& how, cudaStream_t st) {
    const bool scored = a.cap_mul != 0.0f || a.slopes;
    // one token a sequence, at most 8 heads a K/V head (or as few rows in all)
    const bool light = (a.cu_q || a.shared ? (uint64_t)a.tokens * a.group : a.group) <= PR_ROWS / 2;
    if (light) return scored ? launch_rows<T, HD, true, true>(a, how, st) : launch_rows<T, HD, false, true>(a, how, st);
    return scored ? launch_rows<T, HD, true, false>(a, how, st) : launch_rows<T, HD, false, false>(a, how, st);
}

qb200_status pg_rows_launch(const PgArgs& a, int dtype, uint32_t hd, const PgRows& how, cudaStream_t st) {
    if (dtype == QB200_BF16) return hd == 128 ? launch_rows<__nv_bfloat16, 128>(a, how, st) : launch_rows<__nv_bfloat16, 64>(a, how, st);
    return hd == 128 ? launch_rows<__half, 128>(a, how, st) : launch_rows<__half, 64>(a, how, st);
}

}  // namespace qb
