// Paged attention for many rows per K/V head (prompts, chunks of prompts, large groups, a prefix shared by the batch):
// bounded by the tensor pipe and, as closely, by the exponentials (128 x 128 scores cost 1024 cycles of either at head
// dim 128: 4096 multiply-adds and 16 exponentials a cycle and SM).
//
// A unit is 256 (or 128) packed rows of a sequence and one K/V head, over one of `splits` ranges of its keys; one CTA
// each, the longest first (12 prompts of mixed lengths among single tokens: 262 us against 312 with the sequences in the
// order of the batch).  The rows are two tiles of 128 whose steps alternate on the tensor pipe, so that one tile's
// products run under the other's softmax: a prompt of 8192 tokens, 32 / 8 heads of 128, runs at 1.25 PFLOP/s (0.75 of
// measured) in short runs and at 1.05 under the power cap.  A tile's chain bounds it (in cycles: maximum 400,
// exponentials 1350, then P V of the second half and the next Q K^T 1300).  Per step of 128 keys and tile: S = Q K^T (tcgen05.mma, both operands in shared
// memory, accumulator in TMEM), a warpgroup turns S into P (a thread owns a row, so the row's maximum and sum need no
// exchange), P goes back to TMEM over S in the cache's type, and O += P V takes it from there.  The running maximum a
// row's weights are taken against moves only when the true one has passed it by 2^8 (weights then stay below 2^8, far from
// any type's limit), so that the accumulator is rescaled in a few steps of the first tiles and hardly ever after.
//
// P is rounded to the cache's type (half a step of each weight, 2^-8 in bf16, while the row's sum adds the unrounded weights): a
// second product with what the rounding leaves, as the few-rows kernels have it, would make a step's tensor work 1536 cycles
// instead of 1024, where the pipe is the bound.  The errors are independent across keys and of the order of the output's own
// rounding: results differ from the 64-bit definition by 2.0e-3 where rounding alone gives 1.5e-3 (bf16, a prompt of 8192
// tokens), 2.5e-4 and 2.0e-4 in f16, 2.3e-3 and 1.7e-3 behind a shared prefix of 8192 keys.
//
// A block of at most 128 rows uses both warpgroups too: the second takes the odd tiles of keys of the same rows, and
// the two results are joined in shared memory.
//
// Roles: warps 0-3 and 4-7 softmax and epilogue of the two tiles, warp 8 brings K and V tiles by TMA (one box per page
// and 64 columns, 128-byte swizzle), warp 9 issues the products.  All waits are bounded and report through the cache's
// status word.
#include <cuda.h>
#include <string>

#include "paged.cuh"

namespace qb {

// Registers: 384 threads are launched with 168 each (64512 in all); the softmax warpgroups, which hold a row of 128
// scores a thread, take 216, the third one keeps 72.
constexpr uint32_t PP_THREADS = 384, PP_MORE = 216, PP_LESS = 72;
static_assert(2 * PP_MORE + PP_LESS == 3 * 168, "the shares add up to what the launch gets");
constexpr uint32_t PP_KEYS = 128, PP_ROWS = 128;
template <uint32_t HD> struct PpShape {
    static constexpr uint32_t PANEL = 128 * 128;            // 128 rows of 64 elements
    static constexpr uint32_t TILE = PANEL * (HD / 64);     // a Q, K or V tile
    static constexpr uint32_t STAGES = HD == 128 ? 5 : 8;
    static constexpr uint32_t SMEM = 1024 + 2 * TILE + STAGES * TILE + 256;
    static_assert(STAGES * TILE >= 128 * HD * 4 + 1024, "the second warpgroup's result fits the ring");
    static constexpr uint32_t S_COLS = 128, O_COL = 256;    // TMEM: S of tile t at 128 t (P over its first 64), O at 256 + 128 t
};

__device__ __forceinline__ uint32_t pp_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void pp_init(uint64_t* bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(pp_smem(bar)), "r"(count));
}
__device__ __forceinline__ void pp_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pp_smem(bar)) : "memory");
}
__device__ __forceinline__ void pp_expect(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(pp_smem(bar)), "r"(bytes) : "memory");
}
// One thread's bounded wait for a barrier's phase; gives up at once when another role has.
__device__ __forceinline__ bool pp_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* gave_up, uint32_t polls) {
    for (uint32_t i = 0; i < polls; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(pp_smem(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((i & 63u) == 63u && *gave_up) return false;
    }
    *gave_up = 1;
    return false;
}
// The same for a whole warp, which goes on or gives up as one: a lane that went on to the warp's next barrier without those
// that ran out of polls would wait there for good.
__device__ __forceinline__ bool pp_wait_warp(uint64_t* bar, uint32_t parity, volatile uint32_t* gave_up, uint32_t polls) {
    return __all_sync(0xFFFFFFFFu, pp_wait(bar, parity, gave_up, polls));
}
// After giving up: a short wait for what is still in flight.
__device__ __forceinline__ void pp_land(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < 4096; i++) {
        uint32_t ok;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(pp_smem(bar)), "r"(parity) : "memory");
        if (ok) return;
    }
}
__device__ __forceinline__ uint32_t pp_elect() {
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}
__device__ __forceinline__ void pp_load(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, int32_t w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(map),
        "r"(x), "r"(y), "r"(z), "r"(w), "r"(pp_smem(bar))
        : "memory");
}
__device__ __forceinline__ void pp_load3(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(map), "r"(x),
                 "r"(y), "r"(z), "r"(pp_smem(bar))
                 : "memory");
}
// Shared-memory matrix descriptors, 128-byte swizzle.  K-major (Q, K): 8-row groups 1024 bytes apart.  MN-major (V as
// [keys][columns]): groups of 8 keys 1024 bytes apart, panels of 64 columns 16 KB apart.
__device__ __forceinline__ uint64_t pp_desc(uint32_t saddr, uint32_t lead) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void pp_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void pp_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
                 "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void pp_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(pp_smem(bar)) : "memory");
}
__device__ __forceinline__ void pp_tmem_ld32(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void pp_tmem_st32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
        "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void pp_ld_done() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pp_st_done() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pp_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pp_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// (x0, x1) * (m, m) + (c, c)
__device__ __forceinline__ void pp_fma2(float& x0, float& x1, uint64_t m2, uint64_t c2) {
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tfma.rn.f32x2 t, t, %2, %3;\n\tmov.b64 {%0, %1}, t;\n\t}" : "+f"(x0), "+f"(x1) : "l"(m2), "l"(c2));
}
__device__ __forceinline__ void pp_add2(float& x0, float& x1, float y0, float y1) {
    asm("{\n\t.reg .b64 t, u;\n\tmov.b64 t, {%0, %1};\n\tmov.b64 u, {%2, %3};\n\tadd.rn.f32x2 t, t, u;\n\tmov.b64 {%0, %1}, t;\n\t}"
        : "+f"(x0), "+f"(x1) : "f"(y0), "f"(y1));
}
__device__ __forceinline__ uint64_t pp_pack2(float x) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ void pp_mul2(float& x0, float& x1, uint64_t m2) {
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tmul.rn.f32x2 t, t, %2;\n\tmov.b64 {%0, %1}, t;\n\t}" : "+f"(x0), "+f"(x1) : "l"(m2));
}
// tanh(b x) of a pair with |b x| <= 0.3: x (b + u (k0 + k1 u)), u = x^2, with b^3 and b^5 in the coefficients of the
// polynomial that is best there (absolute error 2.9e-7, fitted by reweighted least squares), on the multiply-add pipe: four
// instructions a pair, where the exponential and the reciprocal of the general form would triple the load of the pipe that
// already bounds the softmax.
__device__ __forceinline__ void pp_tanh2(float& x0, float& x1, uint64_t k1, uint64_t k0, uint64_t b) {
    asm("{\n\t.reg .b64 x, u, p;\n\t"
        "mov.b64 x, {%0, %1};\n\t"
        "mul.rn.f32x2 u, x, x;\n\t"
        "fma.rn.f32x2 p, u, %2, %3;\n\t"
        "fma.rn.f32x2 p, p, u, %4;\n\t"
        "mul.rn.f32x2 x, x, p;\n\t"
        "mov.b64 {%0, %1}, x;\n\t}"
        : "+f"(x0), "+f"(x1) : "l"(k1), "l"(k0), "l"(b));
}
// The numbers 0 .. 127 as pairs of floats.
__constant__ uint64_t pp_index[64] = {
    0x3F80000000000000ull, 0x4040000040000000ull, 0x40A0000040800000ull, 0x40E0000040C00000ull, 0x4110000041000000ull,
    0x4130000041200000ull, 0x4150000041400000ull, 0x4170000041600000ull, 0x4188000041800000ull, 0x4198000041900000ull,
    0x41A8000041A00000ull, 0x41B8000041B00000ull, 0x41C8000041C00000ull, 0x41D8000041D00000ull, 0x41E8000041E00000ull,
    0x41F8000041F00000ull, 0x4204000042000000ull, 0x420C000042080000ull, 0x4214000042100000ull, 0x421C000042180000ull,
    0x4224000042200000ull, 0x422C000042280000ull, 0x4234000042300000ull, 0x423C000042380000ull, 0x4244000042400000ull,
    0x424C000042480000ull, 0x4254000042500000ull, 0x425C000042580000ull, 0x4264000042600000ull, 0x426C000042680000ull,
    0x4274000042700000ull, 0x427C000042780000ull, 0x4282000042800000ull, 0x4286000042840000ull, 0x428A000042880000ull,
    0x428E0000428C0000ull, 0x4292000042900000ull, 0x4296000042940000ull, 0x429A000042980000ull, 0x429E0000429C0000ull,
    0x42A2000042A00000ull, 0x42A6000042A40000ull, 0x42AA000042A80000ull, 0x42AE000042AC0000ull, 0x42B2000042B00000ull,
    0x42B6000042B40000ull, 0x42BA000042B80000ull, 0x42BE000042BC0000ull, 0x42C2000042C00000ull, 0x42C6000042C40000ull,
    0x42CA000042C80000ull, 0x42CE000042CC0000ull, 0x42D2000042D00000ull, 0x42D6000042D40000ull, 0x42DA000042D80000ull,
    0x42DE000042DC0000ull, 0x42E2000042E00000ull, 0x42E6000042E40000ull, 0x42EA000042E80000ull, 0x42EE000042EC0000ull,
    0x42F2000042F00000ull, 0x42F6000042F40000ull, 0x42FA000042F80000ull, 0x42FE000042FC0000ull,
};

struct PpArgs {
    PgArgs g;
    uint32_t splits, min_rows, block;  // block: rows of a unit, 256 or 128
    uint32_t q_boxes;  // Q by TMA: 128 rows are a box of whole tokens
    uint32_t polls;    // limit of a wait inside the kernel
    float* parts_acc;  // [splits][tokens * heads][hd] and [splits][tokens * heads][2], splits > 1
    float* parts_ml;
};

__device__ __forceinline__ uint32_t pp_blocks(const PpArgs& a, const PgSeq& s) {
    const uint32_t rows = s.q_len * a.g.group;
    return rows < a.min_rows ? 0 : (rows + a.block - 1) / a.block;
}

template <typename T, uint32_t HD, bool SCORED>
__global__ void __launch_bounds__(PP_THREADS, 1) k_paged_prompt(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                                                                const __grid_constant__ CUtensorMap qmap, const __grid_constant__ PpArgs pa) {
    using S = PpShape<HD>;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sQ = smem;                    // [2][HD / 64 panels][128 rows][128 B]
    uint8_t* sR = sQ + 2 * S::TILE;        // ring of K and V tiles
    uint64_t* full = reinterpret_cast<uint64_t*>(sR + S::STAGES * S::TILE);
    uint64_t* empty = full + S::STAGES;
    uint64_t* q_full = empty + S::STAGES;
    uint64_t* s_full = q_full + 1;         // [2] the tile's S is in TMEM (and every earlier product is complete)
    uint64_t* p_full = s_full + 2;         // [2][2] half of the tile's P (64 keys) is in TMEM
    uint64_t* o_full = p_full + 4;         // [2] the tile's O is complete
    uint64_t* cleaned = o_full + 2;        // the last tile of V has zeros behind its last key
    uint64_t* drained = cleaned + 1;       // after giving up: every product that was issued is complete
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile uint32_t* gave_up = tmem_slot + 1;
    volatile uint32_t* loaded = tmem_slot + 2;  // tiles that were asked for
    const PgArgs& a = pa.g;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // ---- barriers and TMEM (while the lengths travel) ----
    if (tid == 0) {
        for (uint32_t i = 0; i < S::STAGES; i++) {
            pp_init(&full[i], 1);
            pp_init(&empty[i], 1);
        }
        pp_init(q_full, pa.q_boxes ? 1 : 8);
        pp_init(cleaned, 1);
        pp_init(drained, 1);
        for (uint32_t i = 0; i < 2; i++) {
            pp_init(&s_full[i], 1);
            pp_init(&p_full[2 * i], 4);
            pp_init(&p_full[2 * i + 1], 4);
            pp_init(&o_full[i], 1);
        }
        *gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(pp_smem(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pp_before();  // (the barriers of the scan publish all this)
    // ---- which unit: the sequence with the most keys first, in it the last (longest) block first, so that the CTAs that
    // start last have the least to do; batches of more sequences than threads go in their own order ----
    __shared__ uint32_t s_seq, s_before;
    uint64_t* s_kv = reinterpret_cast<uint64_t*>(sQ);  // keys and blocks of the sequences; in the second form block counts of the warps
    __shared__ PgSeq s_found;
    const uint32_t seqs = a.shared ? 1 : a.batch, want = blockIdx.x / (a.kv_heads * pa.splits);
    if (tid == 0) s_seq = 0xFFFFFFFFu;
    if (seqs <= PP_THREADS) {
        PgSeq mine = {};
        uint32_t n = 0;
        uint64_t before = 0;
        if (tid < seqs) {
            mine = pg_seq(a, tid);
            n = pp_blocks(pa, mine);
            s_kv[tid] = (uint64_t)mine.kv << 32 | n;
        }
        __syncthreads();
        if (n) {
#pragma unroll 8
            for (uint32_t i = 0; i < seqs; i++) {
                const uint64_t o = s_kv[i];
                const uint32_t kv = (uint32_t)(o >> 32);
                if (kv > mine.kv || (kv == mine.kv && i < tid)) before += (uint32_t)o;
            }
            if (before <= want && want - before < n) {
                s_seq = tid;
                s_before = (uint32_t)(before + n);
                s_found = mine;
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // Q's copies may land on s_kv next
        __syncthreads();
    } else {
        uint32_t* s_sum = reinterpret_cast<uint32_t*>(s_kv);
        uint64_t before = 0;
        for (uint32_t b0 = 0; b0 < seqs; b0 += PP_THREADS) {
            const uint32_t b = b0 + tid;
            PgSeq mine = {};
            if (b < seqs) mine = pg_seq(a, b);
            const uint32_t n = b < seqs ? pp_blocks(pa, mine) : 0;
            uint32_t incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t t = __shfl_up_sync(0xFFFFFFFFu, incl, o);
                if (lane >= (uint32_t)o) incl += t;
            }
            __syncthreads();
            if (lane == 31) s_sum[warp] = incl;
            __syncthreads();
            uint64_t excl = before + incl - n;
            for (uint32_t i = 0; i < PP_THREADS / 32; i++) {
                if (i < warp) excl += s_sum[i];
                before += s_sum[i];
            }
            if (excl <= want && want - excl < n) {
                s_seq = b;
                s_before = (uint32_t)(excl + n);
                s_found = mine;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncthreads();
            if (s_seq != 0xFFFFFFFFu) break;
        }
    }
    if (s_seq == 0xFFFFFFFFu) {  // the grid is an upper bound (the same for all threads)
        if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(0));
        return;
    }
    pp_after();
    const uint32_t b = s_seq, block = s_before - 1 - want;
    const uint32_t kvh = blockIdx.x / pa.splits % a.kv_heads, split = blockIdx.x % pa.splits;
    const PgSeq sq = s_found;
    const uint32_t all_rows = sq.q_len * a.group, row0 = block * pa.block, rows = min(pa.block, all_rows - row0);
    const uint32_t see = pg_limit(sq, (row0 + rows - 1) / a.group);  // keys the block's last token sees (the most)
    const uint32_t n_all = (see + PP_KEYS - 1) / PP_KEYS;
    const uint32_t t0 = n_all * split / pa.splits, t1 = n_all * (split + 1) / pa.splits, n = t1 - t0;  // (below 2^24 tiles, fewer splits than SMs)
    const bool dual = rows <= PP_ROWS;

    // ---- Q to shared memory.  Where the group divides 128 the loader asks for whole boxes; otherwise row by row, all of it in
    // flight at once, and rows past the last one are zeros (1500 cycles of a unit more).  A unit without keys (a block that sees
    // none, an empty range of a cut one) has no product that would wait for Q: it brings none, since its results go through the
    // same shared memory and nothing may be in flight when the CTA ends ----
    if (!pa.q_boxes && n && warp < 8 && (!dual || warp < 4)) {
        constexpr uint32_t CH = HD / 8, STEP = 128 / CH;
        const uint32_t w = warp >> 2, wt = tid & 127, ch = wt % CH, first = w * PP_ROWS, t_rows = min(PP_ROWS, rows - first);
        const uint32_t whole = STEP / a.group, rest = STEP % a.group;
        uint32_t token = (row0 + first + wt / CH) / a.group, sub = (row0 + first + wt / CH) % a.group;
        const uint16_t* src = static_cast<const uint16_t*>(a.q) + (uint64_t)sq.q0 * a.q_stride + (uint64_t)kvh * a.group * HD + ch * 8;
        const uint32_t dst = pp_smem(sQ) + w * S::TILE + (ch >> 3) * S::PANEL;
#pragma unroll
        for (uint32_t qr = wt / CH; qr < PP_ROWS; qr += STEP) {
            const bool there = qr < t_rows;
            const uint16_t* from = there ? src + (uint64_t)token * a.q_stride + (uint64_t)sub * HD : src;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + qr * 128 + (((ch & 7) ^ (qr & 7)) << 4)), "l"(from), "r"(there ? 16u : 0u) : "memory");
            token += whole;
            sub += rest;
            if (sub >= a.group) {
                sub -= a.group;
                token++;
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    // all 512 columns are this CTA's, so they start at 0; a constant keeps the products' addresses in uniform registers
    constexpr uint32_t tmem = 0;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PP_MORE));
        // ---- softmax and epilogue: warpgroup w owns tile w (or, where the block is one tile, its keys' odd tiles) ----
        const uint32_t w = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t first = dual ? 0 : w * PP_ROWS;  // the tile's first row of the block
        const uint32_t t_rows = min(PP_ROWS, rows - first);
        if (!pa.q_boxes) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) pp_arrive(q_full);
        }

        const uint32_t my = min(r, t_rows - 1);  // a row past the last one runs along with it and is not stored
        const uint32_t row = row0 + first + my, token = row / a.group, head = kvh * a.group + row % a.group;
        const uint32_t lim = pg_limit(sq, token);
        const uint32_t lim_warp = __shfl_sync(0xFFFFFFFFu, lim, 0);  // the warp's least: limits grow with the row
        float slope = 0.0f;
        int32_t pos = 0;
        if (SCORED && a.slopes) {
            slope = a.slopes[head];
            pos = pg_position(a, sq, token);
        }
        const uint32_t t_lane = tmem + (((warp & 3) * 32) << 16);
        const uint32_t t_s = t_lane + w * S::S_COLS, t_o = t_lane + S::O_COL + w * 128;
        // the factor that the exponential still has to apply: cap, or the whole scale of the plain form
        // (a scale that is not positive is applied before)
        const bool before = SCORED && a.cap_mul == 0.0f && !(a.score_mul > 1e-30f);
        const float c = SCORED && a.cap_mul != 0.0f ? a.cap_mul : before ? 1.0f : a.score_mul;
        const uint64_t c2 = pp_pack2(c);
        if (SCORED) slope *= PG_LOG2E / c;  // in units of what the exponential scales
        // 2^8 in units of the score (c is positive).  Q of a row past the last one may be anything (the next sequence's, or
        // nobody's): it has no say in what its warp does, so that nothing of it reaches the others' bits.
        const float slack = r < t_rows ? 8.0f / c : INFINITY;
        float m = -INFINITY, l0 = 0.0f, l1 = 0.0f;
        bool ok = true;
        uint32_t it = 0;
        for (uint32_t t = t0 + (dual ? w : 0); t < t1; t += dual ? 2 : 1, it++) {
            if (!(ok = pp_wait_warp(&s_full[w], it & 1, gave_up, pa.polls))) break;
            pp_after();
            float s[128];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) pp_tmem_ld32(t_s + i * 32, s + i * 32);
            pp_ld_done();
            const uint32_t key0 = t * PP_KEYS;
            float shift = 0.0f;  // of all the row's scores of this tile
            const bool masked = key0 + PP_KEYS > lim_warp;
            const uint32_t left = lim > key0 ? lim - key0 : 0;
            if (SCORED) {
                if (masked && a.cap_mul != 0.0f) {
                    // columns that the row does not see may hold anything (the last tile's, what was in shared memory): they
                    // must not choose the form of the cap
#pragma unroll
                    for (uint32_t i = 0; i < 128; i++) s[i] = i < left ? s[i] : 0.0f;
                }
                if (before) {
                    const uint64_t mul2 = pp_pack2(a.score_mul);
#pragma unroll
                    for (uint32_t i = 0; i < 128; i += 2) pp_mul2(s[i], s[i + 1], mul2);
                }
                if (a.cap_mul != 0.0f) {
                    float far[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (uint32_t i = 0; i < 128; i += 8)
#pragma unroll
                        for (uint32_t k = 0; k < 4; k++) far[k] = fmaxf(fmaxf(far[k], fabsf(s[i + k])), fabsf(s[i + 4 + k]));
                    const float b = a.score_mul;
                    if (__any_sync(0xFFFFFFFFu, slack != INFINITY && !(fmaxf(fmaxf(far[0], far[1]), fmaxf(far[2], far[3])) * fabsf(b) <= 0.3f && fabsf(b) <= 64.0f))) {  // (b^5 stays in range)
#pragma unroll
                        for (uint32_t i = 0; i < 128; i++) s[i] = pg_cap(s[i] * b, 1.0f);
                    } else {
                        const uint64_t k1 = pp_pack2(0.12640675902366638f * b * b * b * b * b), k0 = pp_pack2(-0.33312109112739563f * b * b * b), k = pp_pack2(b);
#pragma unroll
                        for (uint32_t i = 0; i < 128; i += 2) pp_tanh2(s[i], s[i + 1], k1, k0, k);
                    }
                }
                if (a.slopes) {
                    const int32_t d = pos - (int32_t)key0;
                    if (__all_sync(0xFFFFFFFFu, d >= (int32_t)PP_KEYS - 1)) {
                        // no key behind the row's own place: slope * (i - d) for key i, its constant part left to the reference
                        shift = -slope * (float)d;
                        const uint64_t slope2 = pp_pack2(slope);
#pragma unroll
                        for (uint32_t i = 0; i < 128; i += 2)
                            asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%0, %1};\n\tfma.rn.f32x2 t, %2, %3, t;\n\tmov.b64 {%0, %1}, t;\n\t}"
                                : "+f"(s[i]), "+f"(s[i + 1]) : "l"(slope2), "l"(pp_index[i >> 1]));
                    } else {
                        const float d0 = (float)d;
#pragma unroll
                        for (uint32_t i = 0; i < 128; i++) s[i] = fmaf(-slope, fabsf(d0 - (float)i), s[i]);
                    }
                }
            }
            if (masked) {
#pragma unroll
                for (uint32_t i = 0; i < 128; i++) s[i] = i < left ? s[i] : -INFINITY;
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (uint32_t i = 4; i < 124; i += 8)
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) mx[k] = fmaxf(fmaxf(mx[k], s[i + k]), s[i + 4 + k]);  // one three-way maximum
#pragma unroll
            for (uint32_t k = 0; k < 4; k++) mx[k] = fmaxf(mx[k], s[124 + k]);
            const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) + shift;
            if (__any_sync(0xFFFFFFFFu, mt > m + slack)) {
                const float mn = fmaxf(m, mt);
                const float f = m == -INFINITY ? 0.0f : pg_exp2((m - mn) * c);
                m = mn;
                l0 *= f;
                l1 *= f;
                if (it) {  // the products up to the last step are complete: this step's S was issued behind them
#pragma unroll 1
                    for (uint32_t i = 0; i < HD; i += 32) {
                        float o[32];
                        pp_tmem_ld32(t_o + i, o);
                        pp_ld_done();
#pragma unroll
                        for (uint32_t k = 0; k < 32; k++) o[k] *= f;
                        pp_tmem_st32(t_o + i, reinterpret_cast<const uint32_t*>(o));
                    }
                    pp_st_done();
                }
            }
            const uint64_t mc2 = pp_pack2(m == -INFINITY ? 0.0f : (shift - m) * c);
            uint32_t pk[32];
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) {
#pragma unroll
                for (uint32_t i = 0; i < 64; i += 2) {
                    float x0 = s[h * 64 + i], x1 = s[h * 64 + i + 1];
                    pp_fma2(x0, x1, c2, mc2);
                    x0 = pg_exp2(x0);
                    x1 = pg_exp2(x1);
                    pp_add2(l0, l1, x0, x1);
                    pk[i >> 1] = PgType<T>::pack(x0, x1);
                }
                // the product with V begins with the first half while the second one is computed
                pp_tmem_st32(t_s + h * 32, pk);
                pp_st_done();
                pp_before();
                __syncwarp();
                if (lane == 0) pp_arrive(&p_full[2 * w + h]);
            }
        }
        // ---- epilogue ----
        if (ok && it) ok = pp_wait_warp(&o_full[w], 0, gave_up, pa.polls);
        if (ok && dual && w == 1 && n) ok = pp_wait_warp(&o_full[0], 0, gave_up, pa.polls);  // it writes where the other's products read
        pp_after();
        float l = l0 + l1, ml = m * c;  // (-inf stays -inf: c is positive)
        float* other = reinterpret_cast<float*>(sR);  // [HD][128] and then m, l [128] each
        if (dual && w == 1) {
            // its part of the rows, for the first warpgroup; every load of the ring has been read by a product by now
            if (ok && it) {
#pragma unroll 1
                for (uint32_t i = 0; i < HD; i += 32) {
                    float o[32];
                    pp_tmem_ld32(t_o + i, o);
                    pp_ld_done();
#pragma unroll
                    for (uint32_t k = 0; k < 32; k++) other[(i + k) * 128 + r] = o[k];
                }
            }
            if (ok) {
                other[HD * 128 + r] = ml;
                other[HD * 128 + 128 + r] = l;
            }
        }
        if (dual) asm volatile("bar.sync 1, 256;" ::: "memory");
        if (ok && (!dual || w == 0)) {
            float f = 1.0f, g = 0.0f;
            const bool join = dual && n > 1;
            if (join) {
                const float m1 = other[HD * 128 + r], M = fmaxf(ml, m1);
                f = pg_weight(ml, M);
                g = pg_weight(m1, M);
                l = fmaf(l, f, other[HD * 128 + 128 + r] * g);
                ml = M;
            }
            // A thread holds a row, memory wants rows side by side: they go through the warp's share of its Q tile (every
            // product that reads it is complete).  (Stored from the row's own thread, 8 bytes in each of 32 lines an
            // instruction, a unit's output took 7 us.)
            const uint32_t heads = a.group * a.kv_heads, grow = (sq.q0 + token) * heads + head;
            const uint64_t all = (uint64_t)a.tokens * heads;
            const bool parts = pa.splits > 1;
            PgEnd e = {};
            if (r < t_rows) {
                if (parts) *reinterpret_cast<float2*>(pa.parts_ml + (split * all + grow) * 2) = make_float2(ml, l);
                else e = pg_end(a, sq.q0 + token, head, ml, l, true);
            }
            uint8_t* stage = sQ + w * S::TILE + (warp & 3) * (S::TILE / 4);
            const uint32_t n_rows = t_rows > (warp & 3) * 32 ? min(32u, t_rows - (warp & 3) * 32) : 0;
            auto columns = [&](uint32_t from, float (&o)[32]) {  // 32 of the row's columns
                if (it) {
                    pp_tmem_ld32(t_o + from, o);
                    pp_ld_done();
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 32; i++) o[i] = 0.0f;
                }
                if (join) {
#pragma unroll
                    for (uint32_t i = 0; i < 32; i++) o[i] = fmaf(o[i], f, other[(from + i) * 128 + r] * g);
                }
            };
            if (!parts && !a.rows_acc && !a.base_acc) {
                // the call's output: whole rows in its type, 16 bytes a thread
                constexpr uint32_t PER = HD / 8, N = PER;  // threads of a row; rows of each thread (32 * PER / 32)
                const uint32_t row_in = lane / PER, piece = lane % PER;
#pragma unroll 1
                for (uint32_t h = 0; h < HD; h += 32) {
                    float o[32];
                    columns(h, o);
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) {
                        uint4 v;
                        v.x = PgType<T>::pack(o[8 * i] * e.f, o[8 * i + 1] * e.f);
                        v.y = PgType<T>::pack(o[8 * i + 2] * e.f, o[8 * i + 3] * e.f);
                        v.z = PgType<T>::pack(o[8 * i + 4] * e.f, o[8 * i + 5] * e.f);
                        v.w = PgType<T>::pack(o[8 * i + 6] * e.f, o[8 * i + 7] * e.f);
                        *reinterpret_cast<uint4*>(stage + lane * (HD * 2) + (((h / 8 + i) ^ (lane & 7)) << 4)) = v;
                    }
                }
                __syncwarp();
#pragma unroll
                for (uint32_t i0 = 0; i0 < N; i0 += 8) {
                    uint4 v[8];
                    uint32_t to[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) {
                        const uint32_t k = (i0 + i) * (32 / PER) + row_in;
                        v[i] = *reinterpret_cast<const uint4*>(stage + k * (HD * 2) + ((piece ^ (k & 7)) << 4));
                        to[i] = __shfl_sync(0xFFFFFFFFu, grow, k);
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++)
                        if ((i0 + i) * (32 / PER) + row_in < n_rows) *reinterpret_cast<uint4*>(a.out + (uint64_t)to[i] * HD + piece * 8) = v[i];
                }
            } else if (!parts || n) {  // (a range without keys leaves its m and l alone: nothing is read at weight 0)
                // partial results and rows that are joined: 32 bits, half of the columns at a time
                constexpr uint32_t COLS = HD / 2, PER = COLS / 4, N = PER;
                const uint32_t row_in = lane / PER, piece = lane % PER;
#pragma unroll 1
                for (uint32_t h = 0; h < 2; h++) {
                    __syncwarp();
#pragma unroll 1
                    for (uint32_t c0 = 0; c0 < COLS; c0 += 32) {
                        float o[32];
                        columns(h * COLS + c0, o);
#pragma unroll
                        for (uint32_t i = 0; i < 8; i++)
                            *reinterpret_cast<float4*>(stage + lane * (COLS * 4) + (((c0 / 4 + i) ^ (lane & 7)) << 4)) =
                                make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                    }
                    __syncwarp();
#pragma unroll 1
                    for (uint32_t i0 = 0; i0 < N; i0 += 8) {
                        float4 v[8];
                        PgEnd ek[8];
#pragma unroll
                        for (uint32_t i = 0; i < 8; i++) {
                            const uint32_t k = (i0 + i) * (32 / PER) + row_in;
                            v[i] = *reinterpret_cast<const float4*>(stage + k * (COLS * 4) + ((piece ^ (k & 7)) << 4));
                            ek[i].f = __shfl_sync(0xFFFFFFFFu, e.f, k);
                            ek[i].g = __shfl_sync(0xFFFFFFFFu, e.g, k);
                            ek[i].row = __shfl_sync(0xFFFFFFFFu, grow, k);
                        }
#pragma unroll
                        for (uint32_t i = 0; i < 8; i++) {
                            if ((i0 + i) * (32 / PER) + row_in >= n_rows) continue;
                            if (parts) *reinterpret_cast<float4*>(pa.parts_acc + (split * all + ek[i].row) * HD + h * COLS + piece * 4) = v[i];
                            else pg_store4<T, HD>(a, ek[i], h * COLS + piece * 4, v[i]);
                        }
                    }
                }
            }
        }
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(PP_LESS));
      if (warp == 8) {
        // ---- K and V tiles by TMA: K0, then V of a step with K of the next one; in the one-tile form K0, K1 and K of the
        // next but one.  A tile is a box per page (or half a page and less) and 64 columns; pages past the last key that is seen are not read.
        const int32_t* table = a.table + (a.shared ? 0 : (uint64_t)b * a.table_stride);
        const uint32_t ps = 1u << a.ps_log, box = min(ps, PP_KEYS), per = PP_KEYS / box;
        const uint32_t ahead = dual ? 2 : 1;
        uint32_t st = 0, count = 0;
        bool ok = true;
        auto page_of = [&](uint32_t t) -> int32_t {  // lane i: the page of the tile's i-th box
            const uint32_t key = t * PP_KEYS + lane * box;
            if (lane >= per || key >= see) return -1;
            const int32_t p = table[key >> a.ps_log];
            if ((uint32_t)p >= a.n_pages) {
                pg_report(a.status, QB200_ERR_INVALID_PARAM);
                return (int32_t)a.n_pages;  // outside the pool: the copy fills zeros
            }
            return p;
        };
        auto load = [&](const CUtensorMap* map, uint32_t t, int32_t page) {
            if (count >= S::STAGES && !pp_wait_warp(&empty[st], (count / S::STAGES - 1) & 1, gave_up, pa.polls)) { ok = false; return; }
            const uint32_t boxes = min(per, (see - t * PP_KEYS + box - 1) / box);
            if (lane == 0) pp_expect(&full[st], boxes * box * HD * 2);
            __syncwarp();
            if (lane < boxes) {
                const uint32_t key = t * PP_KEYS + lane * box, dst = pp_smem(sR) + st * S::TILE + lane * box * 128;
#pragma unroll
                for (uint32_t p = 0; p < HD / 64; p++)
                    pp_load(dst + p * S::PANEL, map, (int32_t)(p * 64), (int32_t)(key & (ps - 1)), (int32_t)kvh, page, &full[st]);
            }
            count++;
            if (++st == S::STAGES) st = 0;
        };
        if (pa.q_boxes && n && lane == 0) {
            // (rows behind the sequence's last one are the next sequence's, or zeros: their results are not stored)
            const uint32_t tiles = dual ? 1 : 2;
            pp_expect(q_full, tiles * S::TILE);
            for (uint32_t w = 0; w < tiles; w++)
#pragma unroll
                for (uint32_t p = 0; p < HD / 64; p++)
                    pp_load3(pp_smem(sQ) + w * S::TILE + p * S::PANEL, &qmap, (int32_t)(p * 64), (int32_t)(kvh * a.group),
                             (int32_t)(sq.q0 + (row0 + w * PP_ROWS) / a.group), q_full);
        }
        __syncwarp();
        int32_t pages[3];  // of tiles t, t + 1, t + 2
#pragma unroll
        for (uint32_t i = 0; i < 3; i++) pages[i] = i < n ? page_of(t0 + i) : -1;
        if (n) load(&kmap, t0, pages[0]);
        if (ok && ahead == 2 && n > 1) load(&kmap, t0 + 1, pages[1]);
        for (uint32_t i = 0; i < n && ok; i++) {
            load(&vmap, t0 + i, pages[0]);
            if (ok && i + ahead < n) load(&kmap, t0 + i + ahead, dual ? pages[2] : pages[1]);
            pages[0] = pages[1];
            pages[1] = pages[2];
            pages[2] = i + 3 < n ? page_of(t0 + i + 3) : -1;
        }
        if (ok && n && see < t1 * PP_KEYS) {
            // The last tile's rows of V behind the last key that is seen: zeros (their weights are zero, but a page may hold
            // anything there, and 0 * NaN is NaN).  V of the last tile was asked for last; this warp knows its turn of the
            // ring (one that had not followed the ring would take the barrier's earlier turns for it).
            const uint32_t slot = (count - 1) % S::STAGES, valid = see - (t1 - 1) * PP_KEYS;
            if ((ok = pp_wait_warp(&full[slot], ((count - 1) / S::STAGES) & 1, gave_up, pa.polls))) {
                for (uint32_t i = valid * 8 + lane; i < PP_KEYS * 8; i += 32)
#pragma unroll
                    for (uint32_t p = 0; p < HD / 64; p++) *reinterpret_cast<uint4*>(sR + slot * S::TILE + p * S::PANEL + i * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) pp_arrive(cleaned);
            }
        }
        if (lane == 0) *loaded = count;
      } else if (warp == 9 && n) {
        // ---- products: one thread waits and issues (its branches are its own; the operands' addresses are constants but
        // for the ring slot) ----
        if (pp_elect()) {
            constexpr uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
            constexpr uint32_t base = (1u << 4) | (type << 7) | (type << 10) | ((128u >> 4) << 24);
            constexpr uint32_t idesc_s = base | ((PP_KEYS >> 3) << 17), idesc_o = base | (1u << 16) | ((HD >> 3) << 17);
            const uint64_t q_desc = pp_desc(pp_smem(sQ), 16), k_desc = pp_desc(pp_smem(sR), 16), v_desc = pp_desc(pp_smem(sR), S::PANEL);
            auto scores = [&](uint32_t tile, uint32_t q_tile, uint32_t slot) {
                const uint64_t da = q_desc + q_tile * (S::TILE >> 4), db = k_desc + slot * (S::TILE >> 4);
#pragma unroll
                for (uint32_t kk = 0; kk < HD / 16; kk++) {
                    const uint32_t off = (kk >> 2) * (S::PANEL >> 4) + (kk & 3) * 2;
                    pp_mma_ss(tmem + tile * S::S_COLS, da + off, db + off, idesc_s, kk ? 1u : 0u);
                }
                pp_commit(&s_full[tile]);
            };
            auto values = [&](uint32_t tile, uint32_t slot, uint32_t parity, bool more, bool last) -> bool {
                const uint64_t db = v_desc + slot * (S::TILE >> 4);
#pragma unroll
                for (uint32_t h = 0; h < 2; h++) {
                    if (!pp_wait(&p_full[2 * tile + h], parity, gave_up, pa.polls)) return false;
                    pp_after();
#pragma unroll
                    for (uint32_t kk = h * 4; kk < h * 4 + 4; kk++)
                        pp_mma_ts(tmem + S::O_COL + tile * 128, tmem + tile * S::S_COLS + kk * 8, db + kk * (2048 >> 4), idesc_o, (more || kk) ? 1u : 0u);
                }
                if (last) pp_commit(&o_full[tile]);
                return true;
            };
            uint32_t st = 0, par = 0;  // the ring's next tile, in the order they were loaded
            auto next = [&](uint32_t& slot) -> bool {
                slot = st;
                const bool got = pp_wait(&full[st], par, gave_up, pa.polls);
                if (++st == S::STAGES) {
                    st = 0;
                    par ^= 1;
                }
                return got;
            };
            // the last tile of V: the loader clears the rows behind the last key that is seen
            auto next_value = [&](uint32_t i, uint32_t& slot) -> bool {
                if (i + 1 == n && see < (t0 + n) * PP_KEYS && !pp_wait(cleaned, 0, gave_up, pa.polls)) return false;
                return next(slot);
            };
            bool ok = pp_wait(q_full, 0, gave_up, pa.polls);
            uint32_t k_slot = 0, v_slot = 0;
            if (!dual) {
                ok = ok && next(k_slot);
                pp_after();
                if (ok) {
                    scores(0, 0, k_slot);
                    scores(1, 1, k_slot);
                    pp_commit(&empty[k_slot]);
                }
                for (uint32_t i = 0; i < n && ok; i++) {
                    const bool last = i + 1 == n;
                    if (!(ok = next_value(i, v_slot))) break;
                    if (!last && !(ok = next(k_slot))) break;
#pragma unroll
                    for (uint32_t tile = 0; tile < 2; tile++) {
                        if (!(ok = values(tile, v_slot, i & 1, i > 0, last))) break;
                        if (tile == 1 && !last) pp_commit(&empty[v_slot]);  // (nobody waits for the last one)
                        if (!last) scores(tile, tile, k_slot);
                    }
                    if (ok && !last) pp_commit(&empty[k_slot]);
                }
            } else {
                for (uint32_t i = 0; i < 2 && i < n && ok; i++) {
                    if (!(ok = next(k_slot))) break;
                    pp_after();
                    scores(i, 0, k_slot);
                    pp_commit(&empty[k_slot]);
                }
                for (uint32_t i = 0; i < n && ok; i++) {
                    const uint32_t tile = i & 1;
                    if (!(ok = next_value(i, v_slot))) break;
                    if (i + 2 < n && !(ok = next(k_slot))) break;
                    if (!(ok = values(tile, v_slot, (i >> 1) & 1, i > 1, i + 2 >= n))) break;
                    if (i + 1 < n) pp_commit(&empty[v_slot]);
                    if (i + 2 < n) {
                        scores(tile, 0, k_slot);
                        pp_commit(&empty[k_slot]);
                    }
                }
            }
        }
      }
    }
    pp_before();
    __syncthreads();
    if (*gave_up) {
        // Some role has given up, and all have come here: nobody asks for more, but copies that another role would have waited
        // for may be on their way into this memory, and products may read it.  (Without a give-up nothing is in flight: every
        // copy has been waited for by a product, and every product by the epilogue.)
        if (tid == 0) pg_report(a.status, QB200_ERR_TIMEOUT);
        if (warp == 8) {
            const uint32_t count = *loaded;
            for (uint32_t i = count > S::STAGES ? count - S::STAGES : 0; i < count; i++) pp_land(&full[i % S::STAGES], (i / S::STAGES) & 1);
            if (pa.q_boxes && n) pp_land(q_full, 0);
        }
        if (warp == 9 && pp_elect()) {  // the thread that issued them
            pp_commit(drained);
            pp_land(drained, 0);
        }
        __syncthreads();
    }
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// Joins the ranges of keys of every row of the prompt kernel's sequences.
template <typename T, uint32_t HD>
__global__ void __launch_bounds__(128) k_paged_prompt_join(const __grid_constant__ PpArgs pa) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const PgArgs& a = pa.g;
    constexpr uint32_t PER = HD / 4;
    const uint32_t heads = a.group * a.kv_heads;
    const uint64_t all = (uint64_t)a.tokens * heads, row = (uint64_t)blockIdx.x * (128 / PER) + threadIdx.x / PER;
    if (row >= all) return;
    const uint32_t token = (uint32_t)(row / heads), head = (uint32_t)(row % heads), col = (threadIdx.x % PER) * 4;
    if (a.cu_q) {  // is the row one of theirs?  the last b with cu_q[b] <= token
        if ((int32_t)token >= a.cu_q[a.batch]) return;
        if (!a.shared) {
            uint32_t lo = 0, hi = a.batch;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) >> 1;
                if (a.cu_q[mid] <= (int32_t)token) lo = mid; else hi = mid;
            }
            const PgSeq s = pg_seq(a, lo);
            if (token < s.q0 || token - s.q0 >= s.q_len || s.q_len * a.group < pa.min_rows) return;
        }
    }
    float M = -INFINITY, L = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr uint32_t U = 10;  // ranges in flight
#pragma unroll 1
    for (uint32_t i0 = 0; i0 < pa.splits; i0 += U) {
        float2 ml[U];
        float4 e[U];
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const uint64_t i = i0 + u;
            ml[u] = make_float2(-INFINITY, 0.0f);
            if (i0 + u >= pa.splits) continue;
            ml[u] = *reinterpret_cast<const float2*>(pa.parts_ml + (i * all + row) * 2);
            e[u] = *reinterpret_cast<const float4*>(pa.parts_acc + (i * all + row) * HD + col);
        }
        float Mn = M;
#pragma unroll
        for (uint32_t u = 0; u < U; u++) Mn = fmaxf(Mn, ml[u].x);
        const float f = pg_weight(M, Mn);
        M = Mn;
        L *= f;
        v.x *= f;
        v.y *= f;
        v.z *= f;
        v.w *= f;
#pragma unroll
        for (uint32_t u = 0; u < U; u++) {
            const float g = pg_weight(ml[u].x, M);
            if (g == 0.0f) continue;  // no range or no key there (or a weight below the smallest number)
            L = fmaf(ml[u].y, g, L);
            v.x = fmaf(e[u].x, g, v.x);
            v.y = fmaf(e[u].y, g, v.y);
            v.z = fmaf(e[u].z, g, v.z);
            v.w = fmaf(e[u].w, g, v.w);
        }
    }
    pg_emit<T, HD>(a, token, head, col, M, L, v);
}

// ---- host side ---------------------------------------------------------------------------------------------------

// Units that the call can have, over all sequences, with blocks of so many rows.
static uint64_t pp_most_units(const PgArgs& a, uint32_t block) {
    const uint64_t rows = (uint64_t)a.tokens * a.group;
    if (a.shared) return div_ceil(rows, block) * a.kv_heads;
    if (!a.cu_q) return a.batch * div_ceil(a.group, block) * a.kv_heads;
    return (rows / block + (a.batch < a.tokens ? a.batch : a.tokens)) * a.kv_heads;
}

static uint64_t pp_most_keys(const PgArgs& a) { return a.shared ? a.shared : (uint64_t)a.width << a.ps_log; }

// Blocks of one tile of rows for short keys, where all of them fit the SMs at once: more SMs work and fewer partial results
// are joined (us with 128 / 256 rows, 32 / 8 heads: 512 tokens 15.1 / 23.6, 1024 tokens 24.2 / 24.0; 512 tokens against 4000 keys 67 / 51:
// a tile of keys then serves half the rows).
static uint32_t pp_block(const PgArgs& a, uint32_t sms) {
    return pp_most_units(a, PP_ROWS) <= sms && pp_most_keys(a) <= 6 * PP_KEYS ? PP_ROWS : 2 * PP_ROWS;
}

uint32_t pg_prompt_splits(const PgArgs& a, uint32_t sms) {
    // fewer units than SMs: every unit's keys are cut so that all SMs have work, into ranges of at least two tiles
    const uint64_t units = pp_most_units(a, pp_block(a, sms)), keys = pp_most_keys(a);
    const uint64_t by_keys = div_ceil(keys, 2 * PP_KEYS), by_sms = units ? sms / units : 1, s = by_keys < by_sms ? by_keys : by_sms;
    return s > 1 ? (uint32_t)s : 1;
}

uint64_t pg_prompt_part_floats(const PgArgs& a, uint32_t splits, uint32_t hd) {
    return splits > 1 ? (uint64_t)splits * a.tokens * a.group * a.kv_heads * (hd + 2) : 0;
}

typedef CUresult (*PpEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                               const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static PpEncodeFn pp_encode_fn() {
    static PpEncodeFn fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PpEncodeFn>(p);
    }
    return fn;
}

template <typename T, uint32_t HD, bool SCORED>
static qb200_status launch_prompt(const PpArgs& pa, uint32_t grid, const CUtensorMap (&map)[3], cudaStream_t st) {
    static bool attr_set[64] = {};
    int dev = 0;
    QB_CUDA_TRY(cudaGetDevice(&dev));
    if (!attr_set[dev & 63]) {
        QB_CUDA_TRY(cudaFuncSetAttribute(k_paged_prompt<T, HD, SCORED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PpShape<HD>::SMEM));
        attr_set[dev & 63] = true;
    }
    QB_CUDA_TRY(pg_launch(k_paged_prompt<T, HD, SCORED>, dim3(grid), dim3(PP_THREADS), PpShape<HD>::SMEM, st, map[0], map[1], map[2], pa));
    if (pa.splits > 1) {
        const uint64_t rows = (uint64_t)pa.g.tokens * pa.g.group * pa.g.kv_heads, per = 128 / (HD / 4);
        QB_CUDA_TRY(pg_launch(k_paged_prompt_join<T, HD>, dim3((uint32_t)((rows + per - 1) / per)), dim3(128), 0, st, pa));
    }
    return QB200_OK;
}

qb200_status pg_prompt_launch(const PgArgs& a, int dtype, uint32_t hd, uint32_t splits, uint32_t min_rows, cudaStream_t st) {
    PpEncodeFn enc = pp_encode_fn();
    if (!enc) return fail(QB200_ERR_CUDA, "paged attention: cuTensorMapEncodeTiled is not available from this driver");
    int dev = 0;
    QB_CUDA_TRY(cudaGetDevice(&dev));
    const uint32_t ps = 1u << a.ps_log;
    CUtensorMap map[3];
    for (int i = 0; i < 2; i++) {
        const cuuint64_t dims[4] = {hd, ps, a.kv_heads, a.n_pages};
        const cuuint64_t strides[3] = {(cuuint64_t)hd * 2, (cuuint64_t)ps * hd * 2, (cuuint64_t)a.kv_heads * ps * hd * 2};
        const cuuint32_t box[4] = {64, ps < PP_KEYS ? ps : PP_KEYS, 1, 1}, estr[4] = {1, 1, 1, 1};
        const auto encode = [&] {
            return enc(&map[i], dtype == QB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                       const_cast<uint16_t*>(i ? a.v : a.k), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                       CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        };
        CUresult cr = encode();
        if (cr == CUDA_ERROR_INVALID_CONTEXT) {  // a thread without CUDA work so far has no current context until a device is set
            QB_CUDA_TRY(cudaSetDevice(dev));
            cr = encode();
        }
        if (cr != CUDA_SUCCESS) return fail(QB200_ERR_CUDA, "paged attention: cuTensorMapEncodeTiled failed with code " + std::to_string((int)cr));
    }
    PpArgs pa = {};
    pa.g = a;
    map[2] = map[0];  // a valid map either way; unused without boxes
    if (PP_ROWS % a.group == 0) {
        // Q as [tokens][heads][hd]: 128 packed rows are 128 / group tokens of a group's heads
        pa.q_boxes = 1;
        const cuuint64_t dims[3] = {hd, (cuuint64_t)a.group * a.kv_heads, a.tokens}, strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)a.q_stride * 2};
        const cuuint32_t box[3] = {64, a.group, PP_ROWS / a.group}, estr[3] = {1, 1, 1};
        const CUresult cr = enc(&map[2], dtype == QB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(a.q),
                                dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (cr != CUDA_SUCCESS) return fail(QB200_ERR_CUDA, "paged attention: cuTensorMapEncodeTiled (Q) failed with code " + std::to_string((int)cr));
    }
    pa.splits = splits;
    pa.min_rows = min_rows;
    pa.polls = pg_spin_limit();
    pa.parts_acc = a.parts;
    pa.parts_ml = a.parts + (uint64_t)splits * a.tokens * a.group * a.kv_heads * hd;
    uint32_t sms = 0;
    const qb200_status got = pg_sms(&sms);
    if (got) return got;
    pa.block = pp_block(a, sms);
    const uint64_t units = pp_most_units(a, pa.block) * splits;
    if (units > 0x7FFFFFFFull) return fail(QB200_ERR_NOT_SUPPORTED, "paged attention: 2^31 blocks of rows or more");
    const uint32_t grid = (uint32_t)units;
    // a score that is not a positive multiple of q . k takes the general form (the plain one keeps its maximum in q . k)
    const bool scored = a.cap_mul != 0.0f || a.slopes || !(a.score_mul > 1e-30f);
    if (dtype == QB200_BF16) {
        if (hd == 128) return scored ? launch_prompt<__nv_bfloat16, 128, true>(pa, grid, map, st) : launch_prompt<__nv_bfloat16, 128, false>(pa, grid, map, st);
        return scored ? launch_prompt<__nv_bfloat16, 64, true>(pa, grid, map, st) : launch_prompt<__nv_bfloat16, 64, false>(pa, grid, map, st);
    }
    if (hd == 128) return scored ? launch_prompt<__half, 128, true>(pa, grid, map, st) : launch_prompt<__half, 128, false>(pa, grid, map, st);
    return scored ? launch_prompt<__half, 64, true>(pa, grid, map, st) : launch_prompt<__half, 64, false>(pa, grid, map, st);
}

}  // namespace qb
