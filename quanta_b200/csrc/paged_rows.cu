// Paged attention for few rows per K/V head (single tokens, drafts): bounded by the bytes of K and V.
//
// A unit is (sequence of at most 16 packed rows, K/V head); it has ceil(keys / 64) tiles of 64 keys.  The tiles of all
// units, end to end, are cut into equal runs, one per CTA, so that ragged batches and one long sequence keep every SM
// equally busy; a unit cut by a run's end leaves partial results (m, l, acc) that a second kernel joins.  The lengths
// are read on the device, so a captured call follows them.
//
// A CTA has four warps and each takes 16 of a tile's keys on its own: its K and V rows travel by 16-byte asynchronous
// copies through a ring of its own (no barrier in the loop), S = Q K^T and O += P V run on the tensor pipe
// (m16n8k16; the packed rows are the 16) and the softmax is one pass with a running maximum.  The warps' results are
// joined once per unit.  P is rounded to the cache's type for the second product (half a step, 2^-8 in bf16, of each
// weight, while l adds the unrounded weights): the errors are independent across keys and stay below the rounding of
// the output itself.
#include <string>

#include "paged.cuh"

namespace qb {

constexpr uint32_t PR_WARPS = 4, PR_KEYS = 16, PR_TILE = PR_WARPS * PR_KEYS, PR_ROWS = PG_FEW_ROWS;
static_assert(PR_ROWS == 16, "the rows of one tensor instruction");
template <uint32_t HD> struct PrShape {
    static constexpr uint32_t ROW = HD * 2, STAGE = 2 * PR_KEYS * ROW;  // bytes of a row; of a stage (K, then V)
    static constexpr uint32_t STAGES = HD == 128 ? 3 : 6, WARP = STAGES * STAGE, SMEM = PR_WARPS * WARP;
    static constexpr uint32_t ACC = HD + 8;  // floats between rows of the joined accumulator (no bank conflicts)
    static constexpr uint32_t PART = PR_ROWS * (HD + 2);  // floats of one partial result: m, l [16] each, acc [16][hd]
    static_assert(PR_ROWS * ACC * 4 + 2 * PR_ROWS * 4 <= WARP, "a warp's results fit its ring");
};

__device__ __forceinline__ uint32_t pr_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes to shared memory; `bytes` = 0 writes zeros and reads nothing.
__device__ __forceinline__ void pr_copy16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
// where the sequence has more rows than a unit holds (the prompt kernel takes those) or none.
__device__ __forceinline__ uint32_t pr_tiles(const PgSeq& s) { return max(1u, (s.see + PR_TILE - 1) / PR_TILE); }
__device__ __forceinline__ uint64_t pr_weight(const PgArgs& a, const PgSeq& s) {
    const uint64_t rows = (uint64_t)s.q_len * a.group;
    return rows == 0 || rows > PG_FEW_ROWS ? 0 : (uint64_t)a.kv_heads * pr_tiles(s);
}

// Where the CTA's run of tiles lies: [run0, run1) of the total, and the sequence that holds tile run0 (first: its
// first tile).  All threads of the CTA take part.
struct PrRun {
    uint64_t run0, run1, first, total;
    uint32_t seq, ctas;  // CTAs that have a run: none of theirs is empty
};
__device__ __forceinline__ PrRun pr_find_run(const PgArgs& a, uint32_t seqs) {
    __shared__ uint64_t s_warp[PR_WARPS];
    __shared__ uint64_t s_first;
    __shared__ uint32_t s_seq;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint64_t sum = 0, mine = 0;
    for (uint32_t b = tid; b < seqs; b += PR_WARPS * 32) sum += mine = pr_weight(a, pg_seq(a, b));
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) s_warp[warp] = sum;
    if (tid == 0) s_seq = seqs;
    __syncthreads();
    uint64_t total = 0;
#pragma unroll
    for (uint32_t w = 0; w < PR_WARPS; w++) total += s_warp[w];
    PrRun r;
    r.total = total;
    r.ctas = (uint32_t)min((uint64_t)gridDim.x, total);
    r.seq = seqs;
    r.run0 = r.run1 = r.first = 0;
    if (blockIdx.x >= r.ctas) return r;  // the same for all threads of the CTA
    r.run0 = total * blockIdx.x / r.ctas;
    r.run1 = total * (blockIdx.x + 1) / r.ctas;
    uint64_t before = 0;
    for (uint32_t b0 = 0; b0 < seqs; b0 += PR_WARPS * 32) {
        const uint32_t b = b0 + tid;
        const uint64_t w = b < seqs ? (seqs <= PR_WARPS * 32 ? mine : pr_weight(a, pg_seq(a, b))) : 0;
        uint64_t incl = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xFFFFFFFFu, incl, o);
            if (lane >= (uint32_t)o) incl += t;
        }
        __syncthreads();  // s_warp is read by all before it is written again
        if (lane == 31) s_warp[warp] = incl;
        __syncthreads();
        uint64_t excl = before + incl - w;
        for (uint32_t i = 0; i < PR_WARPS; i++) {
            if (i < warp) excl += s_warp[i];
            before += s_warp[i];
        }
        if (excl <= r.run0 && r.run0 < excl + w) {
            s_seq = b;
            s_first = excl;
        }
        __syncthreads();
        if (s_seq < seqs) break;
    }
    r.seq = s_seq;
    r.first = s_first;
    return r;
}

template <typename T, uint32_t HD, bool SCORED>
__global__ void __launch_bounds__(PR_WARPS * 32, 2) k_paged_rows(const PgArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    using S = PrShape<HD>;
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr uint32_t KS = HD / 16, NP = HD / 16, CH = HD / 8;  // k-steps of S, pairs of column tiles of O, 16-byte chunks of a row
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, quad = lane >> 2, part4 = lane & 3;
    const uint32_t seqs = a.shared ? 1 : a.batch;
    const PrRun run = pr_find_run(a, seqs);
    int32_t* meta = a.meta + blockIdx.x * 8;
    if (tid == 0) meta[0] = -1;
    if (run.run0 == run.run1) return;
    uint8_t* ring = smem + warp * S::WARP;
    const uint32_t ring_s = pr_smem(ring);
    uint32_t b = run.seq;
    PgSeq sq = pg_seq(a, b);
    uint64_t seq_first = run.first, at = run.run0;
    uint32_t slot = 0;  // the CTA's first partial unit goes to its slot 0, the last one to slot 1
    while (at < run.run1) {
        while (at >= seq_first + pr_weight(a, sq)) {  // on to the next sequence that has rows here
            seq_first += pr_weight(a, sq);
            if (++b >= seqs) return;
            sq = pg_seq(a, b);
        }
        const uint32_t tiles = pr_tiles(sq), kvh = (uint32_t)((at - seq_first) / tiles);
        const uint64_t unit_first = seq_first + (uint64_t)kvh * tiles;
        const uint32_t t0 = (uint32_t)(at - unit_first);
        const uint32_t t1 = (uint32_t)min((uint64_t)tiles, run.run1 - unit_first);
        at = unit_first + t1;
        const uint32_t rows = sq.q_len * a.group;
        const uint32_t see = pg_limit(sq, sq.q_len - 1);  // keys the last token sees (the most)
        const uint32_t te = min(t1, (see + PR_TILE - 1) / PR_TILE);
        const int32_t* table = a.table + (a.shared ? 0 : (uint64_t)b * a.table_stride);

        // this thread's two rows: what they see, and the bias they get
        uint32_t lim[2];
        float slope[2];
        int32_t pos[2];
        uint32_t qf[KS][4];
        {
            const uint16_t* qp[2] = {nullptr, nullptr};
#pragma unroll
            for (uint32_t i = 0; i < 2; i++) {
                const uint32_t r = quad + 8 * i;
                lim[i] = 0;
                slope[i] = 0.0f;
                pos[i] = 0;
                if (r < rows) {
                    const uint32_t token = r / a.group, head = kvh * a.group + r % a.group;
                    lim[i] = pg_limit(sq, token);
                    qp[i] = static_cast<const uint16_t*>(a.q) + (uint64_t)(sq.q0 + token) * a.q_stride + (uint64_t)head * HD;
                    if (SCORED && a.slopes) {
                        slope[i] = a.slopes[head] * PG_LOG2E;
                        pos[i] = pg_position(a, sq, token);
                    }
                }
            }
#pragma unroll
            for (uint32_t ks = 0; ks < KS; ks++)
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    const uint16_t* p = qp[i & 1];
                    qf[ks][i] = p ? *reinterpret_cast<const uint32_t*>(p + ks * 16 + (i >> 1) * 8 + part4 * 2) : 0u;
                }
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, o[2 * NP][4];
#pragma unroll
        for (uint32_t n = 0; n < 2 * NP; n++) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;

        // the warp's 16 keys of tile t -> a stage of its ring (16-byte chunk c of a row at c ^ (row & 7)); keys that no
        // row sees are zeros, whatever the page holds there, and so are all keys of a page that is not in the pool
        auto fetch = [&](uint32_t t, uint32_t st) {
            const uint32_t key0 = t * PR_TILE + warp * PR_KEYS;
            uint32_t valid = key0 < see ? min(see - key0, PR_KEYS) : 0;
            int32_t page = 0;
            if (valid) {
                page = table[key0 >> a.ps_log];
                if ((uint32_t)page >= a.n_pages) {
                    pg_report(a.status, QB200_ERR_INVALID_PARAM);
                    page = 0;
                    valid = 0;
                }
            }
            const uint64_t base = (((uint64_t)(uint32_t)page * a.kv_heads + kvh) << a.ps_log) + (key0 & ((1u << a.ps_log) - 1));
            const uint32_t dst = ring_s + st * S::STAGE;
#pragma unroll
            for (uint32_t i = 0; i < PR_KEYS * CH / 32; i++) {
                const uint32_t id = i * 32 + lane, row = id / CH, c = id % CH, bytes = row < valid ? 16u : 0u;
                const uint64_t src = (base + (bytes ? row : 0)) * HD + c * 8;
                const uint32_t d = dst + row * S::ROW + ((c ^ (row & 7)) << 4);
                pr_copy16(d, a.k + src, bytes);
                pr_copy16(d + PR_KEYS * S::ROW, a.v + src, bytes);
            }
        };
#pragma unroll
        for (uint32_t i = 0; i + 1 < S::STAGES; i++) {
            if (t0 + i < te) fetch(t0 + i, i);
            pr_commit();
        }
        uint32_t st = 0;
        for (uint32_t t = t0; t < te; t++) {
            pr_wait<S::STAGES - 2>();
            __syncwarp();
            const uint32_t ks_s = ring_s + st * S::STAGE, vs_s = ks_s + PR_KEYS * S::ROW;
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
            const uint32_t key0 = t * PR_TILE + warp * PR_KEYS + part4 * 2;
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (uint32_t n = 0; n < 2; n++)
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    const uint32_t r = i >> 1, key = key0 + n * 8 + (i & 1);
                    float x = s[n][i] * a.score_mul;
                    if (SCORED) {
                        if (a.cap_mul != 0.0f) x = pg_cap(x, a.cap_mul);
                        x = fmaf(-slope[r], fabsf((float)(pos[r] - (int32_t)key)), x);
                    }
                    x = key < lim[r] ? x : -INFINITY;
                    s[n][i] = x;
                    mx[r] = fmaxf(mx[r], x);
                }
            float f[2], ms[2];
#pragma unroll
            for (uint32_t r = 0; r < 2; r++) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xFFFFFFFFu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xFFFFFFFFu, mx[r], 2));
                const float mn = fmaxf(m[r], mx[r]);
                ms[r] = mn == -INFINITY ? 0.0f : mn;
                f[r] = pg_exp2(m[r] - ms[r]);
                m[r] = mn;
                l[r] *= f[r];
            }
            if (__any_sync(0xFFFFFFFFu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
                for (uint32_t n = 0; n < 2 * NP; n++) {
                    o[n][0] *= f[0];
                    o[n][1] *= f[0];
                    o[n][2] *= f[1];
                    o[n][3] *= f[1];
                }
            }
            uint32_t pf[4];
#pragma unroll
            for (uint32_t n = 0; n < 2; n++) {
                float p[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    p[i] = pg_exp2(s[n][i] - ms[i >> 1]);
                    l[i >> 1] += p[i];
                }
                pf[n * 2] = PgType<T>::pack(p[0], p[1]);
                pf[n * 2 + 1] = PgType<T>::pack(p[2], p[3]);
            }
            {
                const uint32_t key = (((lane >> 3) & 1) << 3) | (lane & 7), sub = lane >> 4;
#pragma unroll
                for (uint32_t n = 0; n < NP; n++) {
                    uint32_t vf[4];
                    pr_ldsm_t(vs_s + key * S::ROW + (((n * 2 + sub) ^ (key & 7)) << 4), vf);
                    pr_mma(o[2 * n], pf, vf[0], vf[1], T());
                    pr_mma(o[2 * n + 1], pf, vf[2], vf[3], T());
                }
            }
            __syncwarp();  // every lane is done with the stage that the next fetch overwrites
            {
                const uint32_t tn = t + S::STAGES - 1;
                const uint32_t sn = st == 0 ? S::STAGES - 1 : st - 1;
                if (tn < te) fetch(tn, sn);
                pr_commit();
            }
            if (++st == S::STAGES) st = 0;
        }
        pr_wait<0>();
        __syncwarp();

        // join the warps: each leaves its rows in its own ring
#pragma unroll
        for (uint32_t r = 0; r < 2; r++) {
            l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 1);
            l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], 2);
        }
        float* w_acc = reinterpret_cast<float*>(ring);
        float* w_ml = w_acc + PR_ROWS * S::ACC;
#pragma unroll
        for (uint32_t n = 0; n < 2 * NP; n++) {
            *reinterpret_cast<float2*>(w_acc + quad * S::ACC + n * 8 + part4 * 2) = make_float2(o[n][0], o[n][1]);
            *reinterpret_cast<float2*>(w_acc + (quad + 8) * S::ACC + n * 8 + part4 * 2) = make_float2(o[n][2], o[n][3]);
        }
        if (part4 == 0) {
            w_ml[quad] = m[0];
            w_ml[quad + 8] = m[1];
            w_ml[PR_ROWS + quad] = l[0];
            w_ml[PR_ROWS + quad + 8] = l[1];
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == tiles;
        float* part = a.parts + ((uint64_t)blockIdx.x * 2 + slot) * S::PART;
        if (!whole) {
            // a unit that starts here and goes on: this CTA's entry names what the second kernel joins
            if (tid == 0 && t0 == 0) {
                meta[1] = (int32_t)slot;
                meta[2] = (int32_t)(sq.q0);
                meta[3] = (int32_t)rows;
                meta[4] = (int32_t)kvh;
                // the CTA whose run holds the unit's last tile x: the largest c with total * c / ctas <= x
                meta[0] = (int32_t)(((unit_first + tiles) * run.ctas - 1) / run.total);
            }
        }
        constexpr uint32_t PER = HD / 4;  // threads of a row
        for (uint32_t r = tid / PER; r < rows; r += PR_WARPS * 32 / PER) {
            const uint32_t col = (tid % PER) * 4;
            float M = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < PR_WARPS; w++) M = fmaxf(M, reinterpret_cast<const float*>(smem + w * S::WARP)[PR_ROWS * S::ACC + r]);
            float L = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t w = 0; w < PR_WARPS; w++) {
                const float* p = reinterpret_cast<const float*>(smem + w * S::WARP);
                const float g = pg_weight(p[PR_ROWS * S::ACC + r], M);
                const float4 e = *reinterpret_cast<const float4*>(p + r * S::ACC + col);
                L = fmaf(p[PR_ROWS * S::ACC + PR_ROWS + r], g, L);
                v.x = fmaf(e.x, g, v.x);
                v.y = fmaf(e.y, g, v.y);
                v.z = fmaf(e.z, g, v.z);
                v.w = fmaf(e.w, g, v.w);
            }
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
        slot = 1;
        __syncthreads();  // the rings are free again
    }
}

// Joins the partial results of the unit that starts in CTA blockIdx.x's run and ends in a later one's.  A block takes
// the rows blockIdx.y, blockIdx.y + gridDim.y, ...; LANES groups of threads take every LANES-th part of a row (one
// sequence's keys may be cut into dozens: taken one after the other, 37 parts cost 18 us) and meet in shared memory.
template <typename T, uint32_t HD>
__global__ void __launch_bounds__(256) k_paged_rows_join(const PgArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    using S = PrShape<HD>;
    constexpr uint32_t PER = HD / 4, LANES = 256 / PER, U = 3;
    __shared__ float4 s_acc[LANES][PER];
    __shared__ float s_m[LANES], s_l[LANES];
    const int4 m0 = *reinterpret_cast<const int4*>(a.meta + blockIdx.x * 8);
    if (m0.x < 0) return;
    const uint32_t kvh = (uint32_t)a.meta[blockIdx.x * 8 + 4];
    const uint32_t last = (uint32_t)m0.x, slot0 = (uint32_t)m0.y, q0 = (uint32_t)m0.z, rows = (uint32_t)m0.w;
    const uint32_t lane = threadIdx.x / PER, col = (threadIdx.x % PER) * 4, lanes = min(LANES, last - blockIdx.x + 1);
    for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y) {
        float M = -INFINITY, L = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
        for (uint32_t c0 = blockIdx.x + lane; c0 <= last; c0 += LANES * U) {
            float m[U], l[U];
            float4 e[U];
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                const uint32_t c = min(c0 + u * LANES, last);
                const float* p = a.parts + ((uint64_t)c * 2 + (c == blockIdx.x ? slot0 : 0)) * S::PART;
                m[u] = c0 + u * LANES <= last ? p[r] : -INFINITY;
                l[u] = p[PR_ROWS + r];
                e[u] = *reinterpret_cast<const float4*>(p + 2 * PR_ROWS + r * HD + col);
            }
#pragma unroll
            for (uint32_t u = 0; u < U; u++) {
                if (c0 + u * LANES > last) continue;
                const float Mn = fmaxf(M, m[u]), f = pg_weight(M, Mn), g = pg_weight(m[u], Mn);
                L = fmaf(L, f, l[u] * g);
                v.x = fmaf(v.x, f, e[u].x * g);
                v.y = fmaf(v.y, f, e[u].y * g);
                v.z = fmaf(v.z, f, e[u].z * g);
                v.w = fmaf(v.w, f, e[u].w * g);
                M = Mn;
            }
        }
        s_acc[lane][threadIdx.x % PER] = v;
        if (col == 0) {
            s_m[lane] = M;
            s_l[lane] = L;
        }
        __syncthreads();
        if (lane == 0) {
            for (uint32_t i = 1; i < lanes; i++) {
                const float mi = s_m[i], Mn = fmaxf(M, mi), f = pg_weight(M, Mn), g = pg_weight(mi, Mn);
                const float4 e = s_acc[i][threadIdx.x % PER];
                L = fmaf(L, f, s_l[i] * g);
                v.x = fmaf(v.x, f, e.x * g);
                v.y = fmaf(v.y, f, e.y * g);
                v.z = fmaf(v.z, f, e.z * g);
                v.w = fmaf(v.w, f, e.w * g);
                M = Mn;
            }
            pg_emit<T, HD>(a, q0 + r / a.group, kvh * a.group + r % a.group, col, M, L, v);
        }
        __syncthreads();
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------

uint32_t pg_rows_grid(const PgArgs& a, uint32_t sms) {
    // two CTAs per SM, fewer where the call cannot have as many tiles
    const uint64_t units = a.shared ? 1 : a.batch;
    const uint64_t keys = a.shared ? a.shared : (uint64_t)a.width << a.ps_log;
    const uint64_t most = units * a.kv_heads * (keys ? div_ceil(keys, PR_TILE) : 1);
    return (uint32_t)(most < 2 * sms ? (most ? most : 1) : 2 * sms);
}

uint64_t pg_rows_part_floats(uint32_t grid, uint32_t hd) { return (uint64_t)grid * 2 * PR_ROWS * (hd + 2) + (uint64_t)grid * 8; }

template <typename T, uint32_t HD, bool SCORED>
static qb200_status launch_rows(const PgArgs& a, uint32_t grid, cudaStream_t st) {
    static bool attr_set[64] = {};
    int dev = 0;
    QB_CUDA_TRY(cudaGetDevice(&dev));
    if (!attr_set[dev & 63]) {
        QB_CUDA_TRY(cudaFuncSetAttribute(k_paged_rows<T, HD, SCORED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PrShape<HD>::SMEM));
        attr_set[dev & 63] = true;
    }
    QB_CUDA_TRY(pg_launch(k_paged_rows<T, HD, SCORED>, dim3(grid), dim3(PR_WARPS * 32), PrShape<HD>::SMEM, st, a));
    const uint64_t rows = a.cu_q || a.shared ? (uint64_t)a.tokens * a.group : a.group;
    QB_CUDA_TRY(pg_launch(k_paged_rows_join<T, HD>, dim3(grid, (uint32_t)(rows < 8 ? rows : 8)), dim3(256), 0, st, a));
    return QB200_OK;
}

qb200_status pg_rows_launch(const PgArgs& a, int dtype, uint32_t hd, uint32_t grid, cudaStream_t st) {
    const bool scored = a.cap_mul != 0.0f || a.slopes;
    if (dtype == QB200_BF16) {
        if (hd == 128) return scored ? launch_rows<__nv_bfloat16, 128, true>(a, grid, st) : launch_rows<__nv_bfloat16, 128, false>(a, grid, st);
        return scored ? launch_rows<__nv_bfloat16, 64, true>(a, grid, st) : launch_rows<__nv_bfloat16, 64, false>(a, grid, st);
    }
    if (hd == 128) return scored ? launch_rows<__half, 128, true>(a, grid, st) : launch_rows<__half, 128, false>(a, grid, st);
    return scored ? launch_rows<__half, 64, true>(a, grid, st) : launch_rows<__half, 64, false>(a, grid, st);
}

}  // namespace qb
