// bfloat16 attention of batches whose requests share pages of the cache, on the fifth-generation tensor cores: every shared stretch of keys is attended to by the rows of all its
// requests together.  Compiled for one key and one value head size: -DHEAD_DIM, -DVALUE_DIM (steps of 8 up to 256).
//
// A plan (prefix_plan.cuh) cuts the batch into items: up to 128 rows, rows = (token, query head of the group), against a range of keys that all of them see (a shared stretch) or
// see up to their own position (a request's own keys).  With s_j = c(scale q k_j) - slope (p - j) an item leaves for each of its rows
//   m = max s_j,  l = sum e^(s_j - m),  o = sum e^(s_j - m) v_j          (in powers of two inside)
// and a second kernel merges a token's results in ascending order of their keys:
//   M = max m_i,  out = sum o_i e^(m_i - M) / (sum l_i e^(m_i - M) + e^(sink - M)).
// Scores, m, l and o are 32-bit; the weights e^(s - m) are rounded to bfloat16 for the product with the values (as the engine's other tensor-core attention does: the operands of a
// product have one type, and a relative rounding of 2^-9 a weight is that of the values themselves).
//
// A CTA takes (item, key/value head) pairs off the plan's list, to and fro (the list is sorted, longest first), so that a captured launch serves plans of any number of items.  Roles:
//   warp 0      brings key and value tiles of 128 keys by TMA through the block table of the item's request, box by box of a page, into a ring of stages (the numbers of 32 boxes' pages
//               are read at once and handed out by shuffle: a load of its own for every tile cost it 700 cycles);
//   warp 1      one lane issues tcgen05.mma: S = Q K^T (Q and K from shared memory, M 128, N 128) into one of two score buffers, and O += P V (P from tensor memory, over the
//               scores that it came from; V as it lies in the pages, MN-major).  It is one thread, so its descriptors are additions to precomputed ones (made one by one they cost 100 cycles a
//               product, three times what the tensor core takes);
//   warps 2-3   bring an item's rows of Q into shared memory while the item before is still in its last tiles;
//   warps 4-11  two groups of four, a thread per row: per tile the scores out of tensor memory, mask, exponentials, running maximum and sum, P back; the row of O is scaled again only
//               when its maximum has grown by more than 2^8.
// The two groups take an item's tiles in turn, because one alone spends most of its time on latencies: tile n's maxima need those of tile n - 1, which the other group hands over before
// it begins its exponentials.  Tensor memory: O in columns 0 .. 255 and two score buffers behind it, or, where O has at most 128 columns, three: then the scores of tile n + 2 need not wait for the
// output of tile n, which a group's turn (600 cycles to read and compare 128 scores a row, 1,700 for the exponentials, 350 to hand them over) else has to wait out.
// A warp without rows leaves the tensor core to multiply what lies there: row m of a product depends on row m of its operand alone, and such rows are stored nowhere.
//
// An item of up to 16 rows (a decoding request's own keys) would fill an eighth of such a tile, and its chain of waits (queries, scores, exponentials, output, each a round trip through
// tensor memory) would be as long as a full one's.  There the warps multiply on mma.sync, straight from the ring: a warp takes its share of a tile's keys for the scores and of the values'
// columns for the output, with one barrier a tile in between.  Such items are to run at the rate of the device's memory, 23 bytes a cycle and SM: a tile of 128 keys of 256 (128 KB, 5,600 cycles) is
// worked off by all eight warps in 4,300.  A tile of smaller heads comes faster than one chain of latencies is gone through, so there each group takes every other tile on its own and leaves
// a result of its own (96 requests' own 32,000 keys, heads of 128: 912 us by all warps together, 704 so; heads of 256: 449 and 434, but short items, 8 x 8 on 4,000, 113 and 124).
//
// Head sizes that are no multiple of 64 are widened to one in shared memory: a box copy that reaches past a row's end fills with zeros.  Boxes that hold none of an item's keys are not
// copied; values behind its last key are cleared in shared memory before they are multiplied with their weight of zero (0 x NaN is no zero).
// All waits are bounded; a role that gives up records a code, and every role leaves through the common exit.
#include "tc_common.cuh"
#include "prefix_plan.cuh"

#if !defined(HEAD_DIM) || !defined(VALUE_DIM)
#error "compile with -DHEAD_DIM=<key head size> -DVALUE_DIM=<value head size>"
#endif

constexpr int HD = HEAD_DIM, VD = VALUE_DIM;
static_assert(HD % 8 == 0 && HD >= 8 && HD <= 256 && VD % 8 == 0 && VD >= 8 && VD <= 256, "head sizes in steps of 8 up to 256");
constexpr int VDP = (VD + 63) / 64 * 64;
// (beside values of 256 columns, keys of 192 are worked off in two halves of 128: with stages of 192 columns only three would fit, and four are needed below)
constexpr int HDP = HD > 128 && VDP == 256 ? 256 : (HD + 63) / 64 * 64;
constexpr int BM = 128, BN = 128;
// a stage of the ring: 128 keys of KW columns of K, or VW columns of V
constexpr int KW = HDP == 256 ? 128 : HDP, VW = VDP == 256 ? 128 : VDP;
constexpr int KC = HDP / KW, VC = VDP / VW;
constexpr int STAGE = BN * (KW > VW ? KW : VW) * 2;
constexpr int BUFS = VDP <= 128 ? 3 : 2;           // score buffers
constexpr int THIN = 16;                           // rows of an item that runs on mma.sync
constexpr int Q_BYTES = BM * HDP * 2;
constexpr int SMALL_FIXED = 2 * BM * 4 + BM * 4 + 2 * BM * 4 + 512;      // rows' positions, maxima that the groups hand over, sums of the second group, barriers
// What the warps on a thin item's tile keep: by tile in turn weights [16][128] in bfloat16 and row maxima [16][warps]; sums [warps][16].  It lies behind the queries of 16 rows, the second group's
// behind their second 64 columns; where there are none, both have memory of their own.
constexpr int SIDES = KC == 1 ? 2 : 1, SIDE_WARPS = 8 / SIDES;       // tiles in work at once, warps each
constexpr int THIN_M = 2 * THIN * BN * 2, THIN_L = THIN_M + 2 * THIN * SIDE_WARPS * 4, THIN_BYTES = THIN_L + SIDE_WARPS * THIN * 4;
constexpr bool THIN_APART = HDP == 64;
static_assert(THIN_BYTES <= (BM - THIN) * 128 && THIN_BYTES % 16 == 0, "behind the queries of 16 rows");
constexpr int SMALL = SMALL_FIXED + (THIN_APART ? 2 * THIN_BYTES : 0);
constexpr int MOST_STAGES = (227 * 1024 - Q_BYTES - SMALL) / STAGE;
constexpr int STAGES = MOST_STAGES > 8 ? 8 : MOST_STAGES;
static_assert(STAGES >= 2 && STAGES >= BUFS * VC, "when a tile's scores are there, what its values' stages held before has been used");
constexpr int SMEM = Q_BYTES + STAGES * STAGE + SMALL;
constexpr int THREADS = 128 + 256;
// registers a thread: 168 at the launch; the groups that hold a row's 128 scores take what the other four warps leave (128 x 56 + 256 x 224 <= 384 x 168)
constexpr int REGS_FEW = 56, REGS_MANY = 224;
static_assert(128 * REGS_FEW + 256 * REGS_MANY <= THREADS * 168, "a split of what the launch has");
constexpr int S_COL = BUFS == 3 ? 128 : 256;
constexpr float SLACK = 8.0f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr uint32_t IDESC_S = umma_idesc(BM, BN, false, false), IDESC_PV = umma_idesc(BM, VW, false, true), IDESC_PV_ALL = umma_idesc(BM, VDP, false, true);
enum { GAVE_UP_LOAD = 31, GAVE_UP_MMA = 32, GAVE_UP_SOFTMAX = 33, GAVE_UP_QUERIES = 34, NOT_ALIGNED = 35 };

__device__ __forceinline__ float fast_exp2(float x) {       // ex2.approx: 2 ulp, exp2(-inf) = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// the largest of three
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
    return *reinterpret_cast<float2*>(&d);
}
// 32 bytes at once (a whole sector a thread)
__device__ __forceinline__ void store8(float* to, const uint32_t* v) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
// Products with their operands' descriptors in two halves: the upper one is a constant, an offset is added to the lower one (addresses of shared memory stay below 2^18, so no carry leaves the
// field).  A K-major tile of 128-byte rows, and an MN-major one whose 64-column blocks lie `block` bytes apart, both in groups of eight rows of 1,024 bytes (tc_common.cuh).
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return ((addr >> 4) & 0x3FFF) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_lo_mn(uint32_t addr, uint32_t block) { return ((addr >> 4) & 0x3FFF) | ((block >> 4) << 16); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(DESC_HI) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d), "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(DESC_HI) : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, uint32_t n) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the 256 threads of the groups: true if all of them say so
__device__ __forceinline__ bool all_of_groups(bool ok) {
    uint32_t all;
    asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\tbar.red.and.pred b, 1, 256, a;\n\tselp.u32 %0, 1, 0, b;\n\t}" : "=r"(all) : "r"(ok ? 1u : 0u) : "memory");
    return all != 0;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    const int n = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n));
}

struct Prefix {
    const bf16* q;
    int q_stride;
    const int* block_table;
    int max_pages, nq, nkv, page_size;
    float scale2, capl;                  // both in powers of two
    const float* slopes;
    const int *plan, *items, *tokens;
    int n_items;                         // -1: the plan's header says (a captured step)
    long long rows;                      // results of a kv head
    float *part_o, *part_ml;             // [kv heads][VD / 8][rows][8] (a warp's rows of eight columns are whole lines), [kv heads][rows][2]
    int* status;
};

struct Item { int token, tokens, lo, hi, request, own, row, first; };      // first: the batch's token that it begins with, if the others follow it one by one (else -1)

// Rows r0 .. r0 + 31 (those below `end`) of an item into shared memory, by one warp: queries, positions.
__device__ __forceinline__ void load_rows(const Prefix& p, const Item& item, int g, int rep, int r0, int end, uint32_t q_s, int* at_of) {
    const int lane = threadIdx.x & 31, r = r0 + lane;
    int src = 0;                                                 // in steps of 8 elements
    if (r < end) {
        const int2* t = reinterpret_cast<const int2*>(p.tokens) + item.token + r / rep;
        const int token = item.first >= 0 ? item.first + r / rep : t->x;
        src = token * (p.q_stride / 8) + (g * rep + r % rep) * (HD / 8);
        at_of[r] = t->y;
    }
    constexpr int CH = HDP / 8;                                  // 16-byte pieces of a row: 8 to 32
    const int n = min(32, end - r0);
    for (int i = lane; i - lane < n * CH; i += 32) {
        const int j = i / CH, chunk = i % CH, at = __shfl_sync(0xffffffffu, src, j & 31), rr = r0 + j;
        if (j < n)
            cp_async16(q_s + (chunk >> 3) * (BM * 128) + rr * 128 + (((chunk ^ rr) & 7) << 4), p.q + (chunk < HD / 8 ? (size_t)(at + chunk) * 8 : 0), chunk < HD / 8);
    }
}

__global__ void __launch_bounds__(THREADS, 1)
prefix_kernel(const __grid_constant__ Prefix p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    extern __shared__ __align__(1024) unsigned char smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_addr(smem);
    const uint32_t q_s = base, ring = q_s + Q_BYTES, small = ring + STAGES * STAGE, bars = small + 5 * BM * 4;
    // by score buffer: s_full, p_full, pv_done; by group and warp of it: its maxima are there.  What the tensor core or else the groups' eight warps hand back (stages, queries) counts
    // eight arrivals: the products' thread makes seven of them itself and leaves the last to the products' end.
    const uint32_t full = bars, empty = full + 8 * STAGES, s_full = empty + 8 * STAGES, p_full = s_full + 8 * BUFS, pv_done = p_full + 8 * BUFS, q_full = pv_done + 8 * BUFS,
                   q_empty = q_full + 8, begun = q_empty + 8, o_free = begun + 8, m_ready = o_free + 8, tmem_slot = m_ready + 64;
    int* at_of = reinterpret_cast<int*>(smem + (small - base));                   // [2][128] positions of an item's rows, items in turn
    volatile float* m_of = reinterpret_cast<volatile float*>(at_of + 2 * BM);     // [128]
    volatile float* l_of = m_of + BM;                                             // [2][128] the second group's sums, items in turn
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem + (tmem_slot - base));
    if (base & 1023) {                   // (tiles of swizzled rows begin at multiples of 1,024 bytes)
        if (threadIdx.x == 0) atomicExch(p.status, NOT_ALIGNED);
        return;
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 8); }
        for (int b = 0; b < BUFS; ++b) { mbar_init(s_full + 8 * b, 1); mbar_init(p_full + 8 * b, 4); mbar_init(pv_done + 8 * b, 1); }
        mbar_init(q_full, 2); mbar_init(q_empty, 8);
        mbar_init(begun, 9); mbar_init(o_free, 8);
        for (int i = 0; i < 8; ++i) mbar_init(m_ready + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tc_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot_ptr;

    const int total = (p.n_items >= 0 ? p.n_items : p.plan[PLAN_ITEMS]) * p.nkv;
    const int rep = p.nq / p.nkv, page_shift = 31 - __clz(p.page_size);
    // the CTA's kth pair, to and fro
    auto pair_at = [&](int k) { return k * (int)gridDim.x + ((k & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x); };
    auto item_of = [&](int it) {
        const int4* at = reinterpret_cast<const int4*>(p.items) + (it < total ? it : 0) / p.nkv * 2;
        const int4 a = at[0], b = at[1];
        return Item{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    };
    // The plan was copied before the step's first kernel started: the first item is looked up while the kernel before this one may still run.  (The kernel behind this one starts
    // when its CTAs have left: let go any earlier, the merge's crowd on the SMs that this launch leaves free or is done with first; 64 on 8,192 20.6 us so, 24.4 let go at the roles' ends.)
    Item next = item_of(blockIdx.x);
    pdl_wait();

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEW));
        if (warp == 0) {
            // ---------------- keys and values ----------------
            const int box_rows = p.page_size < BN ? p.page_size : BN, boxes = BN / box_rows, box_shift = 31 - __clz(box_rows);      // boxes of a tile: one to eight
            bool ok = true;
            int fill = 0;
            for (int k = 0, it; ok && (it = pair_at(k)) < total; ++k) {
                const Item item = next;
                next = item_of(pair_at(k + 1));
                const int g = it % p.nkv, lo = item.lo, hi = item.hi, T = (hi - lo + BN - 1) / BN;
                const int* table = p.block_table + (size_t)item.request * p.max_pages;
                // this lane's box of 32 in a row: the row of the pool that it begins with
                auto row_of_box = [&](int window) {
                    const int key = lo + ((window * 32 + lane) << box_shift), index = key >> page_shift;
                    int page = key < hi && index < p.max_pages ? table[index] : 0;
                    if (page < 0) page = 0;
                    return (page * p.nkv + g) * p.page_size + (key & (p.page_size - 1));
                };
                // keys are asked for at most three tiles before the values, so these windows hold both
                int window = 0, before = 0, now = row_of_box(0), later = row_of_box(1);
                auto load = [&](int n, bool value) {
                    const int width = value ? VW : KW, chunks = value ? VC : KC;
                    const int copied = (min(BN, hi - lo - n * BN) + box_rows - 1) >> box_shift;       // boxes that hold keys of the item
                    if (!value && (n * boxes) >> 5 > window) { ++window; before = now; now = later; later = row_of_box(window + 1); }
                    const int box = n * boxes + lane;
                    const int row = __shfl_sync(0xffffffffu, (n * boxes) >> 5 == window ? now : before, box & 31);
                    for (int c = 0; c < chunks; ++c, ++fill) {
                        const int s = fill % STAGES;
                        if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ((fill / STAGES) & 1) ^ 1))) { ok = false; return; }
                        const uint32_t dst = ring + s * STAGE;
                        if (lane == 0) mbar_expect_tx(full + 8 * s, (copied << box_shift) * width * 2);
                        __syncwarp();
                        if (lane < copied)
                            for (int cb = 0; cb < width / 64; ++cb)
                                tma_load_2d(dst + cb * (BN * 128) + (lane << box_shift) * 128, value ? &v_map : &k_map, full + 8 * s, c * width + cb * 64, row);
                    }
                };
                const int ahead = item.tokens * rep <= THIN ? 2 : BUFS;          // (the scores of a thin item's next tile are worked out, or its other group begins, before a tile's output)
                for (int n = 0; n < ahead && n < T && ok; ++n) load(n, false);
                for (int n = 0; n < T && ok; ++n) {
                    load(n, true);
                    if (ok && n + ahead < T) load(n + ahead, false);
                }
            }
            for (int k = 0; k < STAGES && ok; ++k, ++fill)           // nothing in flight at the exit
                if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * (fill % STAGES), ((fill / STAGES) & 1) ^ 1))) ok = false;
            if (!ok) {
                for (int k = fill > STAGES ? fill - STAGES : 0; k < fill; ++k) mbar_wait(full + 8 * (k % STAGES), (k / STAGES) & 1);
                if (lane == 0) atomicExch(p.status, GAVE_UP_LOAD);
            }
            __syncwarp();
        } else if (warp == 1) {
            // ---------------- products ----------------
            if (lane == 0) {
                bool ok = true;
                int use = 0, tile = 0;                               // stages used, tiles begun before this item's
                const uint32_t q_lo = desc_lo(q_s), k_lo = desc_lo(ring), v_lo = desc_lo_mn(ring, BN * 128);
                auto hand_back = [&](uint32_t bar) { mbar_arrive_n(bar, 7); tc_commit(bar); };
                auto scores = [&](int t) -> bool {                   // S = Q K^T of tile t (counted over all items) into its buffer
                    const uint32_t d = tmem + S_COL + t % BUFS * BN;
#pragma unroll
                    for (int c = 0; c < KC; ++c, ++use) {
                        const int s = use % STAGES;
                        if (!mbar_wait(full + 8 * s, (use / STAGES) & 1)) return false;
                        tc_fence_after();
                        const uint32_t kb = k_lo + s * (STAGE >> 4);
#pragma unroll
                        for (int i = 0; i < KW / 16; ++i) {
                            if (c * KW + i * 16 >= HD) continue;     // (columns behind the head's are zeros)
                            const int col = c * (KW / 64) + (i >> 2);
                            mma_ss(d, q_lo + ((col * (BM * 128) + (i & 3) * 32) >> 4), kb + (((i >> 2) * (BN * 128) + (i & 3) * 32) >> 4), IDESC_S, c > 0 || i > 0 ? 1u : 0u);
                        }
                        hand_back(empty + 8 * s);
                    }
                    tc_commit(s_full + 8 * (t % BUFS));
                    return true;
                };
                auto output = [&](int t, bool first) -> bool {       // O += P V
                    if (!mbar_wait(p_full + 8 * (t % BUFS), (t / BUFS) & 1)) return false;
                    const uint32_t pa = tmem + S_COL + t % BUFS * BN;
                    if (VC == 2 && use % STAGES + 1 < STAGES) {      // both halves of the columns side by side in the ring: products of twice the width, the weights read once
                        const int s = use % STAGES;
                        if (!mbar_wait(full + 8 * s, (use / STAGES) & 1) || !mbar_wait(full + 8 * s + 8, ((use + 1) / STAGES) & 1)) return false;
                        tc_fence_after();
                        const uint32_t vb = v_lo + s * (STAGE >> 4);
#pragma unroll
                        for (int i = 0; i < BN / 16; ++i) mma_ts(tmem, pa + i * 8, vb + ((i * (16 * 128)) >> 4), IDESC_PV_ALL, first && i == 0 ? 0u : 1u);
                        hand_back(empty + 8 * s);
                        hand_back(empty + 8 * s + 8);
                        use += 2;
                    } else
#pragma unroll
                    for (int c = 0; c < VC; ++c, ++use) {
                        const int s = use % STAGES;
                        if (!mbar_wait(full + 8 * s, (use / STAGES) & 1)) return false;
                        tc_fence_after();
                        const uint32_t vb = v_lo + s * (STAGE >> 4), d = tmem + c * VW;
#pragma unroll
                        for (int i = 0; i < BN / 16; ++i) mma_ts(d, pa + i * 8, vb + ((i * (16 * 128)) >> 4), IDESC_PV, first && i == 0 ? 0u : 1u);
                        hand_back(empty + 8 * s);
                    }
                    tc_commit(pv_done + 8 * (t % BUFS));
                    return true;
                };
                for (int k = 0; ok && pair_at(k) < total; ++k) {
                    const Item item = next;
                    next = item_of(pair_at(k + 1));
                    const int T = (item.hi - item.lo + BN - 1) / BN;
                    // A wait cannot tell two rounds of a barrier from none.  Thin items go on without this thread, so it has its part in `begun`: the next item's queries come when it has seen this one's.
                    if (!mbar_wait(q_full, k & 1)) { ok = false; break; }
                    mbar_arrive(begun);
                    if (item.tokens * rep <= THIN) {
                        use += T * (KC + VC);
                        continue;
                    }
                    tc_fence_after();
                    // K 0, K 1, (K 2,) V 0, K 2 (3), V 1, ...
                    for (int n = 0; n < BUFS && n < T && ok; ++n) ok = scores(tile + n);
                    if (T <= BUFS) hand_back(q_empty);
                    // The first product with the values waits until the groups have read the outputs of the item before (they began that item when they were through with those before it, and
                    // cannot end this one without the product: the round waited for is the last or the next).
                    if (ok && k > 0) ok = mbar_wait(o_free, (k - 1) & 1);
                    tc_fence_after();
                    for (int n = 0; n < T && ok; ++n) {
                        ok = output(tile + n, n == 0);
                        if (ok && n + BUFS < T) {
                            ok = scores(tile + n + BUFS);
                            if (n + BUFS + 1 == T) hand_back(q_empty);
                        }
                    }
                    tile += T;
                }
                if (!ok) atomicExch(p.status, GAVE_UP_MMA);
            }
        } else {
            // ---------------- queries: a warp takes every other 32 rows (of the first item the groups take them) ----------------
            bool ok = true;
            next = item_of(pair_at(1));
            for (int k = 1, it; (it = pair_at(k)) < total; ++k) {
                const Item item = next;
                next = item_of(pair_at(k + 1));
                const int rows = item.tokens * rep;
                // where they go: the products of the item before have read the queries, its rows' positions of two items ago have been looked up
                if (!__all_sync(0xffffffffu, mbar_wait(q_empty, (k - 1) & 1) && mbar_wait(begun, (k - 1) & 1))) { ok = false; break; }
                for (int r0 = (warp - 2) * 32; r0 < rows; r0 += 64) load_rows(p, item, it % p.nkv, rep, r0, rows, q_s, at_of + (k & 1) * BM);
                asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            if (!ok && lane == 0) atomicExch(p.status, GAVE_UP_QUERIES);
            __syncwarp();
        }
    } else {
        // ---------------- softmax: a thread per row ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_MANY));
        const int group = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
        const uint32_t mine_ready = m_ready + 8 * (group * 4 + quarter), other_ready = m_ready + 8 * ((group ^ 1) * 4 + quarter);
        const float sc = (p.capl > 0.f || p.slopes != nullptr) ? 1.0f : p.scale2;        // capped and biased scores are in powers of two already
        const float pre = p.capl > 0.f ? 1.0f : p.scale2;
        const float cap_in = p.capl > 0.f ? 2.0f * p.scale2 / p.capl : 0.f;
        bool ok = true;
        int use = 0, tile = 0, other_handed = 0;                 // stages used, tiles, maxima that the other group has handed over, before this item
        if ((int)blockIdx.x < total) {                           // the first item's queries: nobody else has anything to do yet
            const int end = min((warp - 3) * 16, next.tokens * rep);
            if ((warp - 4) * 16 < end) load_rows(p, next, (int)blockIdx.x % p.nkv, rep, (warp - 4) * 16, end, q_s, at_of);
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (warp < 6 && lane == 0) mbar_arrive(q_full);
        }
        for (int k = 0, it; (it = pair_at(k)) < total; ++k) {
            const Item item = next;
            next = item_of(pair_at(k + 1));
            const int g = it % p.nkv, lo = item.lo, hi = item.hi, T = (hi - lo + BN - 1) / BN, rows = item.tokens * rep;
            if (!__all_sync(0xffffffffu, mbar_wait(q_full, k & 1))) ok = false;
            if (rows <= THIN) {
                // ---- up to 16 rows: mma.sync; this thread holds parts of rows lane / 4 and lane / 4 + 8 ----
                // A warp weighs its 32 keys of a tile relative to a maximum of its own, rounded up to a whole number: what brings its weights to the maximum of the group's warps is a power
                // of two then, by which bfloat16 weights are multiplied without a rounding when the output's products read them.  So the warps meet once a tile.
                // this warp's blocks of 8 value columns: w * NT ...; its keys in blocks of 16; products of 16 of the head's columns
                constexpr int NT = VDP / 8 / SIDE_WARPS, KB = BN / SIDE_WARPS / 16, STEPS = (HD + 15) / 16;
                static_assert((VW / 8) % NT == 0, "a warp's value columns lie in one stage");
                const int side = SIDES == 2 ? group : 0, w = SIDES == 2 ? quarter : warp - 4, a_row = lane & 15, a_chunk = lane >> 4;
                const int scratch = THIN_APART ? (int)(bars - base) + 512 + side * THIN_BYTES : THIN * 128 + side * (BM * 128);
                uint32_t qf[STEPS][4];
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                    const int c = i * 2 + a_chunk;
                    ldsm4(q_s + (c >> 3) * (BM * 128) + a_row * 128 + (((c ^ a_row) & 7) << 4), qf[i]);
                }
                float o[NT][4], mw[2] = {-INFINITY, -INFINITY}, m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, slope2[2];
                int last[2], pos[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = (lane >> 2) + 8 * i;
                    pos[i] = r < rows ? at_of[(k & 1) * BM + r] : 0;
                    last[i] = r >= rows ? -1 : item.own ? min(pos[i], hi - 1) : hi - 1;
                    slope2[i] = (p.slopes != nullptr && r < rows) ? p.slopes[g * rep + r % rep] * LOG2E : 0.f;
                }
                __syncwarp();
                // The queries are in registers: those of another thin item may come at once.  (A wide one's would overwrite the weights.)
                const bool early = pair_at(k + 1) < total && next.tokens * rep <= THIN;
                if (lane == 0) {
                    mbar_arrive(begun);
                    if (early) mbar_arrive(q_empty);
                }
#pragma unroll
                for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
                volatile float* mx_all = reinterpret_cast<volatile float*>(smem + scratch + THIN_M);
                volatile float* l_all = reinterpret_cast<volatile float*>(smem + scratch + THIN_L);
                const int begin = use;
                // Every warp passes every stage, one by one, and hands each back, the other group's as soon as they are there: a warp that left some out could be overtaken by two rounds of
                // a stage, which a wait cannot tell from none.
                auto landed = [&]() { if (ok && !__all_sync(0xffffffffu, mbar_wait(full + 8 * (use % STAGES), (use / STAGES) & 1))) ok = false; };
                auto handed = [&]() {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty + 8 * (use % STAGES));
                    ++use;
                };
                auto there = [&](int at) {
                    if (SIDES == 2)
                        while (use < at) { landed(); handed(); }
                    landed();
                };
                auto power = [](float d) { return d < -126.f ? 0u : (uint32_t)(127 + (int)d) << 23; };      // 2^d for a whole d <= 0, as the bits of a float
                // the scores of this warp's keys of tile n; stages come as K 0, K 1, V 0, K 2, V 1, ...
                float sv[2 * KB][4];
                auto scores = [&](int n) {
                    float odd[2 * KB][4];                        // (two chains of products a score: steps of 16 columns in turn)
#pragma unroll
                    for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sv[j][e] = odd[j][e] = 0.f;
                    const int k_at = begin + n * KC + max(n - 1, 0) * VC;
#pragma unroll
                    for (int c = 0; c < KC; ++c) {
                        there(k_at + c);
                        const int s = use % STAGES;
                        const uint32_t kb = ring + s * STAGE;
#pragma unroll
                        for (int i0 = 0; i0 < KW / 16; i0 += 4 / KB) {       // (four fragments at once: a load's latency is that of the products behind it)
                            uint32_t b[4 / KB][KB][4];
#pragma unroll
                            for (int u = 0; u < 4 / KB; ++u)
#pragma unroll
                                for (int h = 0; h < KB; ++h) {
                                    if (c * KW + (i0 + u) * 16 >= HD) continue;
                                    const int ka = (i0 + u) * 2 + ((lane >> 3) & 1), b_row = (w * KB + h) * 16 + (lane & 7) + (lane >> 4) * 8;
                                    ldsm4(kb + (ka >> 3) * (BN * 128) + b_row * 128 + (((ka ^ b_row) & 7) << 4), b[u][h]);
                                }
#pragma unroll
                            for (int u = 0; u < 4 / KB; ++u)
#pragma unroll
                                for (int h = 0; h < KB; ++h) {
                                    if (c * KW + (i0 + u) * 16 >= HD) continue;
                                    mma16816(u & 1 ? odd[2 * h] : sv[2 * h], qf[c * (KW / 16) + i0 + u], b[u][h][0], b[u][h][1]);
                                    mma16816(u & 1 ? odd[2 * h + 1] : sv[2 * h + 1], qf[c * (KW / 16) + i0 + u], b[u][h][2], b[u][h][3]);
                                }
                        }
                        handed();
                    }
#pragma unroll
                    for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sv[j][e] += odd[j][e];
                };
                if (SIDES == 1) scores(0);
                for (int n = side; n < T; n += SIDES) {
                    const int key0 = lo + n * BN, turn = (n / SIDES) & 1;
                    const uint32_t p_s = base + scratch + turn * (THIN * BN * 2);
                    if (SIDES == 2) scores(n);
                    const int v_at = begin + min(T, n + 2) * KC + n * VC;
                    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int j = 0; j < 2 * KB; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int i = e >> 1, key = key0 + w * KB * 16 + j * 8 + (lane & 3) * 2 + (e & 1);
                            float x = sv[j][e];
                            if (p.capl > 0.f) x = p.capl * (1.0f - __fdividef(2.0f, 1.0f + __expf(x * cap_in)));
                            else x *= p.scale2;
                            if (p.slopes != nullptr) x = fmaf(-slope2[i], (float)(pos[i] - key), x);
                            sv[j][e] = key <= last[i] ? x : -INFINITY;
                            mx[i] = fmaxf(mx[i], sv[j][e]);
                        }
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = (lane >> 2) + 8 * i;
                        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                        const float top = fmaxf(mw[i], ceilf(mx[i])), from = top == -INFINITY ? 0.f : top;
                        l[i] *= fast_exp2(mw[i] - from);
                        mw[i] = top;
#pragma unroll
                        for (int j = 0; j < 2 * KB; ++j) {
                            const float e0 = fast_exp2(sv[j][2 * i] - from), e1 = fast_exp2(sv[j][2 * i + 1] - from);
                            l[i] += e0 + e1;
                            asm volatile("st.shared.b32 [%0], %1;" ::"r"(p_s + r * (BN * 2) + (((w * 2 * KB + j) ^ (r & 7)) << 4) + (lane & 3) * 4), "r"(pack_bf16(e0, e1)) : "memory");
                        }
                        if ((lane & 3) == 0) mx_all[(turn * THIN + r) * SIDE_WARPS + w] = top;
                    }
                    if (SIDES == 1 && n + 1 < T) scores(n + 1);  // (while the others come to the barrier)
                    if (SIDES == 1 || side == 0) asm volatile("bar.sync 2, %0;" ::"n"(SIDE_WARPS * 32) : "memory");
                    else asm volatile("bar.sync 3, %0;" ::"n"(SIDE_WARPS * 32) : "memory");
                    // this warp's columns of the output
                    uint32_t a[BN / 16][4], f[2][SIDE_WARPS];             // weights; what brings the warps' weights of the two rows to one reference, twice in a register
#pragma unroll
                    for (int i = 0; i < BN / 16; ++i) ldsm4(p_s + a_row * (BN * 2) + (((i * 2 + a_chunk) ^ (a_row & 7)) << 4), a[i]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float4* of_row = reinterpret_cast<const float4*>(smem + scratch + THIN_M) + (turn * THIN + (lane >> 2) + 8 * i) * (SIDE_WARPS / 4);
                        float mj[SIDE_WARPS], top = m[i];
#pragma unroll
                        for (int j = 0; j < SIDE_WARPS / 4; ++j) {
                            const float4 u = of_row[j];
                            mj[4 * j] = u.x; mj[4 * j + 1] = u.y; mj[4 * j + 2] = u.z; mj[4 * j + 3] = u.w;
                            top = max3(top, fmaxf(u.x, u.y), fmaxf(u.z, u.w));
                        }
                        const float from = top == -INFINITY ? 0.f : top, corr = __uint_as_float(power(m[i] - from));
                        m[i] = top;
#pragma unroll
                        for (int j = 0; j < SIDE_WARPS; ++j) { const uint32_t x = power(mj[j] - from); f[i][j] = __byte_perm(x, x, 0x3232); }
#pragma unroll
                        for (int j = 0; j < NT; ++j) { o[j][2 * i] *= corr; o[j][2 * i + 1] *= corr; }
                    }
#pragma unroll
                    for (int i = 0; i < BN / 16; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const __nv_bfloat162 v = __hmul2(*reinterpret_cast<__nv_bfloat162*>(&a[i][e]), *reinterpret_cast<__nv_bfloat162*>(&f[e & 1][i / KB]));
                            a[i][e] = *reinterpret_cast<const uint32_t*>(&v);
                        }
#pragma unroll
                    for (int c = 0; c < VC; ++c) {
                        there(v_at + c);
                        const int s = use % STAGES, col0 = w * NT - c * (VW / 8);      // the first block's place in this chunk
                        if (col0 >= 0 && col0 < VW / 8) {
                            const uint32_t vb = ring + s * STAGE;
                            if (key0 + BN > hi) {                // (slots behind the last key hold whatever lay there: 0 x NaN is no zero)
                                for (int r = hi - key0 + lane; r < BN; r += 32)
#pragma unroll
                                    for (int j = 0; j < NT; ++j)
                                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vb + ((col0 + j) >> 3) * (BN * 128) + r * 128 + ((((col0 + j) ^ r) & 7) << 4)), "r"(0u)
                                                     : "memory");
                                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // (the stage's next tile comes by TMA: not before these)
                                __syncwarp();
                            }
#pragma unroll
                            for (int i = 0; i < BN / 16; i += 2) {
                                uint32_t b[NT][4];
                                const int key = i * 16 + lane;
#pragma unroll
                                for (int j = 0; j < NT; ++j) ldsm4t(vb + ((col0 + j) >> 3) * (BN * 128) + key * 128 + ((((col0 + j) ^ key) & 7) << 4), b[j]);
#pragma unroll
                                for (int j = 0; j < NT; ++j) mma16816(o[j], a[i], b[j][0], b[j][1]);
#pragma unroll
                                for (int j = 0; j < NT; ++j) mma16816(o[j], a[i + 1], b[j][2], b[j][3]);
                            }
                        }
                        handed();
                    }
                }
                while (use < begin + T * (KC + VC)) { landed(); handed(); }
                // (The second group without a tile leaves no result: its sums are read by nobody, and a warp that stored them here could overtake the one that still reads the item before's,
                // which only a tile's barrier holds back.)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
                    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
                    if ((lane & 3) == 0 && (side == 0 || T > 1)) l_all[w * THIN + (lane >> 2) + 8 * i] = l[i] * __uint_as_float(power(mw[i] - (m[i] == -INFINITY ? 0.f : m[i])));
                }
                if (!all_of_groups(ok)) {
                    if (!ok) atomicExch(p.status, GAVE_UP_SOFTMAX);
                    break;
                }
                if (side == 0 || T > 1) {                        // (the second group's results lie behind the first's)
                    const int row0 = item.row + side * rows;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int r = (lane >> 2) + 8 * i;
                        if (w == 0 && (lane & 3) == 0 && r < rows) {
                            float sum = 0.f;
#pragma unroll
                            for (int j = 0; j < SIDE_WARPS; ++j) sum += l_all[j * THIN + r];
                            *reinterpret_cast<float2*>(p.part_ml + ((size_t)g * p.rows + row0 + r) * 2) = make_float2(m[i], sum);
                        }
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            const int col = w * NT + j;
                            if (r < rows && col < VD / 8)
                                *reinterpret_cast<float2*>(p.part_o + (((size_t)g * (VD / 8) + col) * p.rows + row0 + r) * 8 + (lane & 3) * 2) = make_float2(o[j][2 * i], o[j][2 * i + 1]);
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) {
                    if (!early) mbar_arrive(q_empty);
                    mbar_arrive(o_free);
                }
                continue;
            }
            const bool live = row < rows, warp_live = row - lane < rows;
            const int pos = live ? at_of[(k & 1) * BM + row] : 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(begun);
            const int last = item.own ? min(pos, hi - 1) : hi - 1;         // the last key that the row sees
            const float slope2 = (p.slopes != nullptr && live) ? p.slopes[g * rep + row % rep] * LOG2E : 0.f;
            float m_run = -INFINITY, l_run = 0.f;                          // m_run: what l_run is relative to
            for (int n = group; ok && n < T; n += 2) {
                const int key0 = lo + n * BN, t = tile + n;
                const uint32_t scores_at = t_lane + S_COL + t % BUFS * BN;
                if (!__all_sync(0xffffffffu, mbar_wait(s_full + 8 * (t % BUFS), (t / BUFS) & 1))) { ok = false; break; }
                // (the maxima up to tile n - 1 are the other group's; its P V comes before this one's)
                float corr = 1.f;
                bool changed = false;
                if (warp_live) {
                    tc_fence_after();
                    uint32_t sv[4][32];
#pragma unroll
                    for (int h = 0; h < 4; ++h) tc_ld32(scores_at + 32 * h, sv[h]);
                    tc_wait_ld();
                    if (p.capl > 0.f) {      // tanh(x) = 1 - 2 / (1 + e^(2x)), x = score * scale / cap
#pragma unroll
                        for (int c = 0; c < BN; ++c)
                            sv[c >> 5][c & 31] = __float_as_uint(p.capl * (1.0f - __fdividef(2.0f, 1.0f + __expf(__uint_as_float(sv[c >> 5][c & 31]) * cap_in))));
                    }
                    if (p.slopes != nullptr) {
#pragma unroll
                        for (int c = 0; c < BN; ++c)
                            sv[c >> 5][c & 31] = __float_as_uint(fmaf(-slope2, (float)(pos - (key0 + c)), __uint_as_float(sv[c >> 5][c & 31]) * pre));
                    }
                    if (!__all_sync(0xffffffffu, !live || key0 + BN - 1 <= last)) {
#pragma unroll
                        for (int c = 0; c < BN; ++c) sv[c >> 5][c & 31] = key0 + c <= last ? sv[c >> 5][c & 31] : __float_as_uint(-INFINITY);
                    }
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < BN; c += 2) mx4[(c >> 1) & 3] = max3(mx4[(c >> 1) & 3], __uint_as_float(sv[c >> 5][c & 31]), __uint_as_float(sv[c >> 5][(c & 31) + 1]));
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                    float m_before = -INFINITY;
                    if (n > 0) {
                        if (!__all_sync(0xffffffffu, mbar_wait(other_ready, (other_handed + (n - 1) / 2) & 1))) { ok = false; break; }
                        m_before = m_of[row];
                    }
                    const float m_tile = fmaxf(m_before, mx * sc);
                    const float m_new = m_tile > m_before + SLACK ? m_tile : m_before;     // m_before = -inf: takes m_tile
                    m_of[row] = m_new;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(mine_ready);
                    const float mbase = m_new == -INFINITY ? 0.f : m_new;
                    corr = fast_exp2(m_before - mbase);
                    l_run *= fast_exp2(m_run - mbase);
                    m_run = m_new;
                    changed = live && m_new > m_before;
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    const float2 sc2 = make_float2(sc, sc), minus = make_float2(-mbase, -mbase);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t packed[32];
#pragma unroll
                        for (int c = 0; c < 64; c += 2) {
                            const int at = h * 64 + c;
                            const float2 x = fma2(make_float2(__uint_as_float(sv[at >> 5][at & 31]), __uint_as_float(sv[at >> 5][(at & 31) + 1])), sc2, minus);
                            const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                            sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], e);
                            packed[c >> 1] = pack_bf16(e.x, e.y);
                        }
                        tc_st32(scores_at + 32 * h, packed);
                    }
                    const float2 both = add2(sum[0], sum[1]);
                    l_run += both.x + both.y;
                }
                // O holds the products of all tiles before this one: it is scaled when they are complete
                if (n > 0 && __any_sync(0xffffffffu, changed)) {
                    if (!__all_sync(0xffffffffu, mbar_wait(pv_done + 8 * ((t - 1) % BUFS), ((t - 1) / BUFS) & 1))) { ok = false; break; }
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < VDP; c0 += 32) {
                        uint32_t ov[32];
                        tc_ld32(t_lane + c0, ov);
                        tc_wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * corr);
                        tc_st32(t_lane + c0, ov);
                    }
                }
                // Behind the item's last key the tile holds whatever lay there; its weights are zeros, but 0 x NaN is no zero.  The values' stages are not handed back before this
                // tile's output, and what was in them before has been used (the scores of this tile come behind it).
                if (key0 + BN > hi) {
                    const int first = use + min(T, n + BUFS) * KC + n * VC, held = hi - key0;
                    bool there = true;
                    for (int c = 0; c < VC; ++c) {
                        const int s = (first + c) % STAGES;
                        there = there && mbar_wait(full + 8 * s, ((first + c) / STAGES) & 1);
                        for (int i = row; i < (BN - held) * (VW / 8); i += 128) {
                            const int r = held + i / (VW / 8), rest = i % (VW / 8);
                            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(ring + s * STAGE + (rest >> 3) * (BN * 128) + r * 128 + (rest & 7) * 16), "r"(0u) : "memory");
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    if (!__all_sync(0xffffffffu, there)) { ok = false; break; }
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * (t % BUFS));
            }
            // the last product of the item (every one before it is complete then), by the group that it belongs to
            const int end = tile + T - 1;
            const bool ends = ((T - 1) & 1) == group;
            if (ok && ends && !__all_sync(0xffffffffu, mbar_wait(pv_done + 8 * (end % BUFS), (end / BUFS) & 1))) ok = false;
            if (group == 1) {                            // the second group's sum, relative to the last maximum
                float m = m_run;
                if (ok && !ends && warp_live) {
                    if (!__all_sync(0xffffffffu, mbar_wait(other_ready, (other_handed + (T - 1) / 2) & 1))) ok = false;
                    m = m_of[row];
                }
                l_of[(k & 1) * BM + row] = l_run * fast_exp2(m_run - (m == -INFINITY ? 0.f : m));
            }
            tile += T;
            use += T * (KC + VC);
            if (warp_live) other_handed += group == 0 ? T / 2 : (T + 1) / 2;
            if (!all_of_groups(ok)) {                    // they go on or give up together
                if (!ok) atomicExch(p.status, GAVE_UP_SOFTMAX);
                break;
            }
            if (warp_live) {
                tc_fence_after();
                const size_t at = (size_t)item.row + row;
                if (live && group == 0) {
                    const float m = m_of[row], l = l_run * fast_exp2(m_run - (m == -INFINITY ? 0.f : m)) + l_of[(k & 1) * BM + row];
                    *reinterpret_cast<float2*>(p.part_ml + ((size_t)g * p.rows + at) * 2) = make_float2(m, l);
                }
                // each group stores half the columns
                constexpr int HALF = (VD + 63) / 64 * 32;
#pragma unroll 1
                for (int c0 = group * HALF; c0 < min(VD, group * HALF + HALF); c0 += 32) {
                    uint32_t ov[32];
                    tc_ld32(t_lane + c0, ov);
                    tc_wait_ld();
                    if (live)
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
                            if (c0 + c < VD) store8(p.part_o + (((size_t)g * (VD / 8) + (c0 + c) / 8) * p.rows + at) * 8, ov + c);
                }
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tc_dealloc(tmem, 512);
    }
}

// The merge of a token's results: grid (tokens, kv heads, groups of warps).  A warp's lanes are up to four neighbouring query heads, whose rows of eight columns are one line, by `split` results,
// by blocks of eight columns: lane i of those that share a row's block takes results i, i + split, ..., eight at a time, with a running maximum, and what they have is added up by shuffles.  (No
// shared memory: that would keep the next launch, which wants all of an SM's, from getting ready meanwhile.)  Bound by the latency of its chain of loads (starts, list, results), hence the
// eight in flight, and the more lanes a row the fewer rows there are (8 heads of 256 by one lane, and so: 2 tokens of 65 results 11.7 and 5.8 us, 64 of 19 6.0 and 4.9).
constexpr int MERGE_WARPS = 4, MERGE_SPLIT = 8;
__host__ __device__ __forceinline__ int merge_heads(int rep) { return rep >= 4 ? 4 : rep >= 2 ? 2 : 1; }
__host__ __device__ __forceinline__ int merge_units(int rep, int split) {
    const int heads = merge_heads(rep), blocks = 32 / (heads * split);
    return (rep + heads - 1) / heads * ((VD / 8 + blocks - 1) / blocks);
}
__global__ void __launch_bounds__(MERGE_WARPS * 32)
prefix_merge_kernel(bf16* __restrict__ out, int out_stride, const int* __restrict__ plan, int rep, long long rows, const float* __restrict__ part_o, const float* __restrict__ part_ml,
                    const float* __restrict__ sinks, int split) {
    pdl_wait();
    const int token = blockIdx.x, g = blockIdx.y, unit = (int)blockIdx.z * MERGE_WARPS + (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (unit >= merge_units(rep, split)) return;
    const int heads = merge_heads(rep), groups = (rep + heads - 1) / heads, part = lane / heads % split;
    const int h = unit % groups * heads + lane % heads, col = unit / groups * (32 / (heads * split)) + lane / (heads * split);
    const bool live = h < rep && col < VD / 8;
    const int* starts = plan + plan[PLAN_AT_STARTS];
    const int first = starts[token], n = starts[token + 1] - first;
    const int* list = plan + plan[PLAN_AT_RESULTS] + first;
    const float* mine_o = part_o + ((size_t)g * (VD / 8) + col) * rows * 8;
    const float2* mine_ml = reinterpret_cast<const float2*>(part_ml) + (size_t)g * rows;
    float M = -INFINITY, L = 0.f, O[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    constexpr int AHEAD = 8;
    for (int i0 = part; live && i0 < n; i0 += AHEAD * split) {
        float4 v[AHEAD][2];
        float2 ml[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            ml[u] = make_float2(-INFINITY, 0.f);
            if (i0 + u * split < n) {
                const size_t at = (size_t)list[i0 + u * split] + h;
                ml[u] = mine_ml[at];
                v[u][0] = reinterpret_cast<const float4*>(mine_o + at * 8)[0];
                v[u][1] = reinterpret_cast<const float4*>(mine_o + at * 8)[1];
            }
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) top = fmaxf(top, ml[u].x);
        const float base = top == -INFINITY ? 0.f : top, keep = exp2f(M - base);
        M = top;
        L *= keep;
#pragma unroll
        for (int j = 0; j < 8; ++j) O[j] *= keep;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const float f = exp2f(ml[u].x - base);
            if (i0 + u * split < n) {
                L = fmaf(ml[u].y, f, L);
                O[0] = fmaf(v[u][0].x, f, O[0]); O[1] = fmaf(v[u][0].y, f, O[1]); O[2] = fmaf(v[u][0].z, f, O[2]); O[3] = fmaf(v[u][0].w, f, O[3]);
                O[4] = fmaf(v[u][1].x, f, O[4]); O[5] = fmaf(v[u][1].y, f, O[5]); O[6] = fmaf(v[u][1].z, f, O[6]); O[7] = fmaf(v[u][1].w, f, O[7]);
            }
        }
    }
    pdl_launch_dependents();       // (at the start it cost 96 requests' layer 3 us: the next launch's CTAs came to lie unevenly beside this one's)
    for (int o = heads; o < heads * split; o *= 2) {
        const float other = __shfl_xor_sync(0xffffffffu, M, o), top = fmaxf(M, other), base = top == -INFINITY ? 0.f : top, keep = exp2f(M - base);
        M = top;
        L *= keep;
        L += __shfl_xor_sync(0xffffffffu, L, o);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            O[j] *= keep;
            O[j] += __shfl_xor_sync(0xffffffffu, O[j], o);
        }
    }
    if (!live || n <= 0 || part > 0) return;
    if (sinks) L += exp2f(sinks[g * rep + h] * LOG2E - (M == -INFINITY ? 0.f : M));
    const float inv = 1.0f / L;
    bf16* to = out + (size_t)token * out_stride + (size_t)(g * rep + h) * VD + col * 8;
    *reinterpret_cast<uint2*>(to) = uint2{pack_bf16(O[0] * inv, O[1] * inv), pack_bf16(O[2] * inv, O[3] * inv)};
    *reinterpret_cast<uint2*>(to + 4) = uint2{pack_bf16(O[4] * inv, O[5] * inv), pack_bf16(O[6] * inv, O[7] * inv)};
}

// --------------------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------------------
typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiled encoder() {
    static EncodeTiled fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = reinterpret_cast<EncodeTiled>(p);
    }
    return fn;
}
// A pool [pages][nkv][page_size][head] as a matrix of rows x head; boxes of box_rows x 64 columns, 128-byte swizzle, zeros past a row's end.  (The map is a function of what is
// encoded in it; it is made anew for every launch.)
static int pool_map(const void* ptr, long long rows, int box_rows, int head, CUtensorMap* out) {
    EncodeTiled enc = encoder();
    if (!enc) return 6;
    const cuuint64_t dims[2] = {(cuuint64_t)head, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)head * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, elem[2] = {1, 1};
    const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? WLLM_OK : 2000 + (int)r;
}

// The attention of a planned batch.  pool_pages: pages of the pools; n_tokens: rows of q and out; scratch: nkv * rows * (VD + 2) floats, rows as the plan has them (or the most that a plan of
// this array may have); items_at, tokens_at: their places in the plan; n_items: its items, or -1: its header says; pairs: (item, kv head) pairs, or the most that there may be; ctas: SMs.  sinks, slopes: 32-bit [nq] or null; cap > 0: scores become cap tanh(score / cap).
WLLM_API int wllm_prefix_attention(const void* q, int q_stride, void* out, int out_stride, const void* k_pages, const void* v_pages, long long pool_pages, const int* block_table,
                                   int max_pages, int n_tokens, int nq, int nkv, int page_size, float scale, float cap, const float* sinks, const float* slopes, const int* plan,
                                   int items_at, int tokens_at, int n_items, float* scratch, long long rows, long long pairs, int ctas, int* status, cudaStream_t stream) {
    if (n_tokens <= 0 || pairs <= 0) return WLLM_OK;
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0 || nq / nkv > BM || page_size < 16 || (page_size & (page_size - 1)) || pool_pages < 1 || max_pages < 1 || nkv > 65535 || ctas < 1 ||
        !(scale > 0.f) || !(cap >= 0.f) || rows < 1 || items_at < 0 || tokens_at < 0 || pool_pages * nkv > 0x7fffffffLL / page_size ||
        (long long)n_tokens * (q_stride / 8) > 0x7fffffffLL)
        return WLLM_BAD_SIZE;
    if (q_stride % 8 != 0 || out_stride % 4 != 0 || ((uintptr_t)q & 15) || ((uintptr_t)out & 7) || ((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15) || ((uintptr_t)scratch & 31) || ((uintptr_t)plan & 15) || items_at % 4 != 0 || tokens_at % 2 != 0)
        return WLLM_BAD_ALIGN;
    CUtensorMap km, vm;
    const int box = page_size < BN ? page_size : BN;
    int r = pool_map(k_pages, pool_pages * nkv * page_size, box, HD, &km);
    if (r) return r;
    r = pool_map(v_pages, pool_pages * nkv * page_size, box, VD, &vm);
    if (r) return r;
    static bool configured = false;
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(prefix_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return 1000 + (int)e;
        configured = true;
    }
    Prefix p;
    p.q = (const bf16*)q; p.q_stride = q_stride; p.block_table = block_table; p.max_pages = max_pages; p.nq = nq; p.nkv = nkv; p.page_size = page_size;
    p.scale2 = scale * LOG2E; p.capl = cap * LOG2E; p.slopes = slopes; p.plan = plan; p.items = plan + items_at; p.tokens = plan + tokens_at; p.n_items = n_items; p.rows = rows; p.status = status;
    p.part_o = scratch; p.part_ml = scratch + (size_t)nkv * rows * VD;
    const int st = wllm_launch(prefix_kernel, dim3((unsigned)(pairs < ctas ? pairs : ctas)), THREADS, SMEM, stream, p, km, vm);
    if (st) return st;
    const int rep = nq / nkv;
    // lanes that share a row's block: as many as keep the device's SMs at 16 warps each
    int split = 1;
    while (split < MERGE_SPLIT && (long long)n_tokens * nkv * merge_units(rep, 2 * split) <= 16LL * ctas) split *= 2;
    return wllm_launch(prefix_merge_kernel, dim3(n_tokens, nkv, (merge_units(rep, split) + MERGE_WARPS - 1) / MERGE_WARPS), MERGE_WARPS * 32, 0, stream, (bf16*)out, out_stride, plan, rep, rows,
                       (const float*)p.part_o, (const float*)p.part_ml, sinks, split);
}
