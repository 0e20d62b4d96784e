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
//   warp 0      brings key and value tiles of 128 keys by TMA through the block table of the item's request, box by box of a page, into a ring of stages;
//   warp 1      one lane issues tcgen05.mma: S = Q K^T (Q and K from shared memory, M 128, N 128) into one of two score buffers, and O += P V (P from tensor memory, over the
//               scores that it came from; V as it lies in the pages, MN-major);
//   warps 4-11  two groups of four, a thread per row: the rows of Q into shared memory, then per tile the scores out of tensor memory, mask, exponentials, running maximum and sum, P
//               back; the row of O is scaled again only when its maximum has grown by more than 2^8.
// Two groups, because one alone spends most of its time on latencies: a tile's exponentials are 1,024 cycles of the SM's special function units, a group took 2.3 times that.  An item of more than
// 128 rows gives each group 128 rows of its own (value heads of up to 128, whose two outputs fit tensor memory; the keys come into shared memory once for both).  In an item of up to 128
// rows the groups take its tiles in turn: tile n's maxima need those of tile n - 1, which the other group hands over before it begins its exponentials.
// A warp without rows leaves the tensor core to multiply what lies there: row m of a product depends on row m of its operand alone, and such rows are stored nowhere.
// Tensor memory: O (of the first group's rows, of the second's behind it) in columns 0 .. 255, the score buffers at 256 and 384.
//
// Head sizes that are no multiple of 64 are widened to one in shared memory: a box copy that reaches past a row's end fills with zeros.  Boxes that hold none of an item's keys are not
// copied; values behind its last key are cleared in shared memory before they are multiplied with their weight of zero (0 x NaN is no zero).
// All waits are bounded; a role that gives up records a code, and every role leaves through the common exit.
#include "tc_common.cuh"
#include "prefix_plan.cuh"

#include <mutex>
#include <unordered_map>

#if !defined(HEAD_DIM) || !defined(VALUE_DIM)
#error "compile with -DHEAD_DIM=<key head size> -DVALUE_DIM=<value head size>"
#endif

constexpr int HD = HEAD_DIM, VD = VALUE_DIM;
static_assert(HD % 8 == 0 && HD >= 8 && HD <= 256 && VD % 8 == 0 && VD >= 8 && VD <= 256, "head sizes in steps of 8 up to 256");
constexpr int HDP = (HD + 63) / 64 * 64, VDP = (VD + 63) / 64 * 64;
constexpr int BM = 128, BN = 128;
// a stage of the ring: 128 keys of KW columns of K, or VW columns of V
constexpr int KW = HDP == 256 ? 128 : HDP, VW = VDP == 256 ? 128 : VDP;
constexpr int KC = HDP / KW, VC = VDP / VW;
constexpr int STAGE = BN * (KW > VW ? KW : VW) * 2;
// groups of 128 rows that an item may have: two where both outputs fit tensor memory and both groups' queries leave the ring room for several tiles
constexpr int GROUPS = VDP <= 128 && HDP <= 128 ? 2 : 1;
constexpr int ROWS = GROUPS * BM;
constexpr int Q_BYTES = BM * HDP * 2;              // of one group of rows
constexpr int SMALL = ROWS * 8 + BM * 4 + 512;      // rows' places, maxima that the groups hand over, barriers
constexpr int MOST_STAGES = (227 * 1024 - 1024 - GROUPS * Q_BYTES - SMALL) / STAGE;
constexpr int STAGES = MOST_STAGES > 8 ? 8 : MOST_STAGES;
static_assert(STAGES >= KC + VC || GROUPS == 1, "a tile's keys are in use while the values of the one before are");
static_assert(STAGES >= 2, "a stage for keys and one for values");
constexpr int SMEM = 1024 + GROUPS * Q_BYTES + STAGES * STAGE + SMALL;
constexpr int THREADS = 128 + 256;
// registers a thread: 168 at the launch; the groups that hold a row's 128 scores take what the other four warps leave (128 x 80 + 256 x 208 <= 384 x 168)
constexpr int REGS_FEW = 80, REGS_MANY = 208;
static_assert(128 * REGS_FEW + 256 * REGS_MANY <= THREADS * 168, "a split of what the launch has");
constexpr int S_COL = 256;
constexpr float SLACK = 8.0f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr uint32_t IDESC_S = umma_idesc(BM, BN, false, false), IDESC_PV = umma_idesc(BM, VW, false, true);
enum { GAVE_UP_LOAD = 31, GAVE_UP_MMA = 32, GAVE_UP_SOFTMAX = 33 };

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
    float *part_o, *part_ml;             // [kv heads][rows][VD], [kv heads][rows][2]
    int* status;
};

__global__ void __launch_bounds__(THREADS, 1)
prefix_kernel(const __grid_constant__ Prefix p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    extern __shared__ unsigned char smem_raw[];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_s = base, ring = q_s + GROUPS * Q_BYTES, rows_s = ring + STAGES * STAGE, bars = rows_s + ROWS * 8 + BM * 4;
    // by score buffer: s_full, p_full, pv_done; by group and warp of it: its maxima are there
    const uint32_t full = bars, empty = full + 8 * STAGES, s_full = empty + 8 * STAGES, p_full = s_full + 16, pv_done = p_full + 16, q_full = pv_done + 16, edge_full = q_full + 8,
                   m_ready = edge_full + 8, tmem_slot = m_ready + 64;
    unsigned char* smem = smem_raw + (base - smem_addr(smem_raw));
    struct Row { int src, at; };                             // a row's place in q (in steps of 8 elements), its position
    Row* row_of = reinterpret_cast<Row*>(smem + (rows_s - base));
    // an item's rows are looked up at its beginning; at its end the second group leaves its maximum and sum of a row in the row's place
    volatile float* second = reinterpret_cast<volatile float*>(row_of);
    volatile float* m_of = reinterpret_cast<volatile float*>(row_of + ROWS);
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem + (tmem_slot - base));

    const int total = (p.n_items >= 0 ? p.n_items : p.plan[PLAN_ITEMS]) * p.nkv;
    const int rep = p.nq / p.nkv, page_shift = 31 - __clz(p.page_size);
    // the CTA's kth pair; the last one lies past the end
    auto pair_at = [&](int k) { return k * (int)gridDim.x + ((k & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x); };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(s_full + 8 * b, 1); mbar_init(p_full + 8 * b, 4); mbar_init(pv_done + 8 * b, 1); }
        mbar_init(q_full, 8);
        mbar_init(edge_full, 1);
        for (int i = 0; i < 8; ++i) mbar_init(m_ready + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tc_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot_ptr;

    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_FEW));
    if (warp == 0) {
        // ---------------- keys and values ----------------
        const int box_rows = p.page_size < BN ? p.page_size : BN;
        bool ok = true;
        int fill = 0, edges = 0;
        auto load = [&](const int* table, int g, int key0, int key_hi, bool value) {
            const int width = value ? VW : KW, chunks = value ? VC : KC;
            const int held = min(BN, key_hi - key0), copied = (held + box_rows - 1) / box_rows * box_rows;      // rows of keys, rows that are copied
            const bool edge = value && held < BN;
            // this lane's box (pages of 16 or more: at most eight of a tile)
            int row0 = 0;
            if (lane * box_rows < copied) {
                const int key = key0 + lane * box_rows, index = key >> page_shift;
                int page = index < p.max_pages ? table[index] : 0;
                if (page < 0) page = 0;
                row0 = (page * p.nkv + g) * p.page_size + (key & (p.page_size - 1));
            }
            for (int c = 0; c < chunks; ++c) {
                const int s = fill % STAGES;
                if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ((fill / STAGES) & 1) ^ 1))) { ok = false; return; }
                const uint32_t dst = ring + s * STAGE;
                // values that reach past the item's last key land on a barrier of their own, are cleared there, and are announced then
                const uint32_t bar = edge ? edge_full : full + 8 * s;
                if (lane == 0) mbar_expect_tx(bar, copied * width * 2);
                __syncwarp();
                if (lane * box_rows < copied)
                    for (int cb = 0; cb < width / 64; ++cb)
                        tma_load_2d(dst + cb * (BN * 128) + lane * box_rows * 128, value ? &v_map : &k_map, bar, c * width + cb * 64, row0);
                if (edge) {
                    if (!__all_sync(0xffffffffu, mbar_wait(edge_full, edges & 1))) { ok = false; return; }
                    ++edges;
                    for (int i = lane; i < (BN - held) * (VW / 8); i += 32) {
                        const int row = held + i / (VW / 8), rest = i % (VW / 8);
                        asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(dst + (rest >> 3) * (BN * 128) + row * 128 + (rest & 7) * 16), "r"(0u) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + 8 * s);
                }
                ++fill;
            }
        };
        for (int k = 0, it; ok && (it = pair_at(k)) < total; ++k) {
            const int* item = p.items + (it / p.nkv) * PLAN_ITEM;
            const int g = it % p.nkv, lo = item[ITEM_KEY_LO], hi = item[ITEM_KEY_HI], T = (hi - lo + BN - 1) / BN;
            const bool two = item[ITEM_TOKENS] * rep > BM;
            const int* table = p.block_table + (size_t)item[ITEM_REQUEST] * p.max_pages;
            const int ahead = two ? 1 : 2;                       // keys are asked for that many tiles before the values
            for (int n = 0; n < ahead && n < T && ok; ++n) load(table, g, lo + n * BN, hi, false);
            for (int n = 0; n < T && ok; ++n) {
                load(table, g, lo + n * BN, hi, true);
                if (ok && n + ahead < T) load(table, g, lo + (n + ahead) * BN, hi, false);
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
            int use = 0, done = 0;                               // stages used, items
            int turn[2] = {0, 0};                                // uses of the score buffers
            // S = Q K^T of rows `rows_at` with the tile whose first stage is `at`, into buffer b; `last`: the stages are free behind it
            auto scores = [&](int at, int group, int b, bool wait, bool last) -> bool {
                for (int c = 0; c < KC; ++c) {
                    const int s = (at + c) % STAGES;
                    if (wait && !mbar_wait(full + 8 * s, ((at + c) / STAGES) & 1)) return false;
                    tc_fence_after();
                    const uint32_t kb = ring + s * STAGE, qb = q_s + group * Q_BYTES;
                    const int steps = min(KW, HD - c * KW + 15) / 16;          // (columns behind the head's are zeros)
                    for (int k = 0; k < steps; ++k) {
                        const int col = c * (KW / 64) + (k >> 2);
                        tc_mma(tmem + S_COL + b * BN, smem_desc(qb + col * (BM * 128) + (k & 3) * 32), smem_desc(kb + (k >> 2) * (BN * 128) + (k & 3) * 32), IDESC_S, c > 0 || k > 0 ? 1u : 0u);
                    }
                    if (last) tc_commit(empty + 8 * s);
                }
                tc_commit(s_full + 8 * b);
                return true;
            };
            auto output = [&](int at, int group, int b, bool first, bool wait, bool last) -> bool {
                if (!mbar_wait(p_full + 8 * b, turn[b] & 1)) return false;
                ++turn[b];
                const uint32_t pa = tmem + S_COL + b * BN;
                for (int c = 0; c < VC; ++c) {
                    const int s = (at + c) % STAGES;
                    if (wait && !mbar_wait(full + 8 * s, ((at + c) / STAGES) & 1)) return false;
                    tc_fence_after();
                    const uint32_t vb = ring + s * STAGE;
#pragma unroll
                    for (int k = 0; k < BN / 16; ++k)
                        tc_mma_ts(tmem + group * VDP + c * VW, pa + k * 8, smem_desc_mn(vb + k * (16 * 128), BN * 128), IDESC_PV, first && k == 0 ? 0u : 1u);
                    if (last) tc_commit(empty + 8 * s);
                }
                tc_commit(pv_done + 8 * b);
                return true;
            };
            for (int k = 0, it; ok && (it = pair_at(k)) < total; ++k, ++done) {
                const int* item = p.items + (it / p.nkv) * PLAN_ITEM;
                const int T = (item[ITEM_KEY_HI] - item[ITEM_KEY_LO] + BN - 1) / BN;
                if (!mbar_wait(q_full, done & 1)) { ok = false; break; }
                tc_fence_after();
                if (GROUPS == 2 && item[ITEM_TOKENS] * rep > BM) {
                    // both groups' rows against each tile: K 0, V 0, K 1, V 1, ...
                    ok = scores(use, 0, 0, true, false) && scores(use, 1, 1, false, true);
                    use += KC;
                    for (int n = 0; n < T && ok; ++n) {
                        const int v = use, next = use + VC;
                        ok = output(v, 0, 0, n == 0, true, false);
                        if (ok && n + 1 < T) ok = scores(next, 0, 0, true, false);
                        ok = ok && output(v, 1, 1, n == 0, false, true);
                        if (ok && n + 1 < T) ok = scores(next, 1, 1, false, true);
                        use += VC + (n + 1 < T ? KC : 0);
                    }
                } else {
                    // tiles in turn: K 0, K 1, V 0, K 2, V 1, ...
                    for (int n = 0; n < 2 && n < T && ok; ++n, use += KC) ok = scores(use, 0, n, true, true);
                    for (int n = 0; n < T && ok; ++n) {
                        ok = output(use, 0, n & 1, n == 0, true, true);
                        use += VC;
                        if (ok && n + 2 < T) {
                            ok = scores(use, 0, n & 1, true, true);
                            use += KC;
                        }
                    }
                }
            }
            if (!ok) atomicExch(p.status, GAVE_UP_MMA);
        }
    }
    } else {
        // ---------------- softmax: a thread per row ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_MANY));
        const int group = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane, tid = threadIdx.x - 128;
        const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16), scores_at = t_lane + S_COL + group * BN;
        const uint32_t mine_ready = m_ready + 8 * (group * 4 + quarter), other_ready = m_ready + 8 * ((group ^ 1) * 4 + quarter);
        const float sc = (p.capl > 0.f || p.slopes != nullptr) ? 1.0f : p.scale2;        // capped and biased scores are in powers of two already
        const float pre = p.capl > 0.f ? 1.0f : p.scale2;
        const float cap_in = p.capl > 0.f ? 2.0f * p.scale2 / p.capl : 0.f;
        bool ok = true;
        int turn = 0, other_turn = 0, other_handed = 0;          // uses of this group's score buffer, of the other's, maxima that the other has handed over, before this item
        for (int k = 0, it; (it = pair_at(k)) < total; ++k) {
            const int* item = p.items + (it / p.nkv) * PLAN_ITEM;
            const int g = it % p.nkv, lo = item[ITEM_KEY_LO], hi = item[ITEM_KEY_HI], T = (hi - lo + BN - 1) / BN, rows = item[ITEM_TOKENS] * rep;
            const bool own = item[ITEM_OWN] != 0, two = rows > BM;
            const int m_row = two ? group * BM + row : row;
            const bool live = m_row < rows, warp_live = m_row - lane < rows;
            if (m_row < rows && (two || group == 0)) {
                const int* t = p.tokens + 2 * (item[ITEM_TOKEN] + m_row / rep);
                row_of[m_row] = Row{t[0] * (p.q_stride / 8) + (g * rep + m_row % rep) * (HD / 8), t[1]};
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            for (int i = tid; i < rows * (HDP / 8); i += 256) {
                const int r = i / (HDP / 8), chunk = i % (HDP / 8);
                cp_async16(q_s + (r >> 7) * Q_BYTES + (chunk >> 3) * (BM * 128) + (r & 127) * 128 + (((chunk ^ r) & 7) << 4), p.q + (chunk < HD / 8 ? (size_t)(row_of[r].src + chunk) * 8 : 0),
                           chunk < HD / 8);
            }
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            const int pos = live ? row_of[m_row].at : 0;
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            asm volatile("bar.sync 1, 256;" ::: "memory");                 // nobody looks a row up any more: `second` may be written
            const int last = own ? min(pos, hi - 1) : hi - 1;              // the last key that the row sees
            const float slope2 = (p.slopes != nullptr && live) ? p.slopes[g * rep + m_row % rep] * LOG2E : 0.f;
            const uint32_t o_at = t_lane + (two ? group * VDP : 0);
            float m_run = -INFINITY, l_run = 0.f;                          // m_run: what l_run is relative to
            for (int n = two ? 0 : group; n < T; n += two ? 1 : 2, ++turn) {
                const int key0 = lo + n * BN;
                if (!__all_sync(0xffffffffu, mbar_wait(s_full + 8 * group, turn & 1))) { ok = false; break; }
                // tiles in turn: the maxima up to tile n - 1 are the other group's; its P V comes before this one's
                const bool behind = !two && n > 0;
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
                    float m_before = m_run;
                    if (behind) {
                        if (!__all_sync(0xffffffffu, mbar_wait(other_ready, (other_handed + (n - 1) / 2) & 1))) { ok = false; break; }
                        m_before = m_of[row];
                    }
                    const float m_tile = fmaxf(m_before, mx * sc);
                    const float m_new = m_tile > m_before + SLACK ? m_tile : m_before;     // m_before = -inf: takes m_tile
                    if (!two) {
                        m_of[row] = m_new;
                        __syncwarp();
                        if (lane == 0) mbar_arrive(mine_ready);
                    }
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
                    const bool there = two ? mbar_wait(pv_done + 8 * group, (turn - 1) & 1) : mbar_wait(pv_done + 8 * (group ^ 1), (other_turn + (n - 1) / 2) & 1);
                    if (!__all_sync(0xffffffffu, there)) { ok = false; break; }
                    tc_fence_after();
#pragma unroll 1
                    for (int c0 = 0; c0 < VDP; c0 += 32) {
                        uint32_t ov[32];
                        tc_ld32(o_at + c0, ov);
                        tc_wait_ld();
#pragma unroll
                        for (int c = 0; c < 32; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * corr);
                        tc_st32(o_at + c0, ov);
                    }
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * group);
            }
            // the last product of the item (every one before it is complete then), by the group that it belongs to
            if (ok && (two || ((T - 1) & 1) == group) && !__all_sync(0xffffffffu, mbar_wait(pv_done + 8 * group, (turn - 1) & 1))) ok = false;
            const int others = two ? T : group == 0 ? T / 2 : (T + 1) / 2;
            other_turn += others;
            if (!two && warp_live) other_handed += others;
            if (!two && group == 1) { second[2 * row] = m_run; second[2 * row + 1] = l_run; }
            uint32_t all;                                // they go on or give up together
            asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\tbar.red.and.pred b, 1, 256, a;\n\tselp.u32 %0, 1, 0, b;\n\t}" : "=r"(all) : "r"(ok ? 1u : 0u) : "memory");
            if (!all) {
                if (!ok) atomicExch(p.status, GAVE_UP_SOFTMAX);
                break;
            }
            if (warp_live) {
                tc_fence_after();
                const size_t at = (size_t)g * p.rows + item[ITEM_ROW] + m_row;
                if (live && (two || group == 0)) {
                    float m = m_run, l = l_run;
                    if (!two) {
                        m = m_of[row];
                        const float mbase = m == -INFINITY ? 0.f : m;
                        l = l_run * fast_exp2(m_run - mbase) + second[2 * row + 1] * fast_exp2(second[2 * row] - mbase);
                    }
                    *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
                }
                // of an item of up to 128 rows each group stores half the columns
                constexpr int HALF = (VD + 63) / 64 * 32;
                const int c_lo = two ? 0 : group * HALF, c_hi = two ? VD : min(VD, c_lo + HALF);
#pragma unroll 1
                for (int c0 = c_lo; c0 < c_hi; c0 += 32) {
                    uint32_t ov[32];
                    tc_ld32(o_at + c0, ov);
                    tc_wait_ld();
                    if (live)
#pragma unroll
                        for (int c = 0; c < 32; c += 8)
                            if (c0 + c < VD) store8(p.part_o + at * VD + c0 + c, ov + c);
                }
                tc_fence_before();                       // read before the next item's products are let loose on O (by q_full)
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tc_dealloc(tmem, 512);
    }
}

// The merge of a token's results: grid (tokens, kv heads, groups of warps), a warp per (query head, 128 columns).  Bound by the latency of its chain of loads (starts, list, maxima and sums,
// results) where results are few, so a unit's loads are asked for eight at a time and every unit has a warp of its own.
constexpr int MERGE_WARPS = 4, MERGE_BLOCKS = (VD + 127) / 128;
__global__ void __launch_bounds__(MERGE_WARPS * 32)
prefix_merge_kernel(bf16* __restrict__ out, int out_stride, const int* __restrict__ plan, int rep, long long rows, const float* __restrict__ part_o, const float* __restrict__ part_ml,
                    const float* __restrict__ sinks) {
    pdl_begin();
    const int token = blockIdx.x, g = blockIdx.y, unit = (int)blockIdx.z * MERGE_WARPS + (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (unit >= rep * MERGE_BLOCKS) return;
    const int* starts = plan + plan[PLAN_AT_STARTS];
    const int first = starts[token], n = starts[token + 1] - first;
    if (n <= 0) return;
    const int* list = plan + plan[PLAN_AT_RESULTS] + first;
    const size_t head0 = (size_t)g * rows;
    const int h = unit / MERGE_BLOCKS, col = (unit % MERGE_BLOCKS) * 128 + lane * 4, head = g * rep + h;
    float M = -INFINITY, L = 0.f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < n; i0 += 32) {
        const size_t row = i0 + lane < n ? head0 + list[i0 + lane] + h : 0;
        const float2 ml = i0 + lane < n ? *reinterpret_cast<const float2*>(part_ml + row * 2) : make_float2(-INFINITY, 0.f);
        const int count = min(32, n - i0);
        float keep = 1.f, mine = 0.f;
        for (int u0 = 0; u0 < count; u0 += 8) {
            float4 v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const size_t at = __shfl_sync(0xffffffffu, row, (u0 + u) & 31);
                v[u] = u0 + u < count && col < VD ? *reinterpret_cast<const float4*>(part_o + at * VD + col) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            if (u0 == 0) {                       // while they are on their way
                const float M_new = fmaxf(M, warp_max(ml.x)), base = M_new == -INFINITY ? 0.f : M_new;
                keep = exp2f(M - base);
                mine = exp2f(ml.x - base);
                L = L * keep + warp_sum(ml.y * mine);
                O.x *= keep; O.y *= keep; O.z *= keep; O.w *= keep;
                M = M_new;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float f = __shfl_sync(0xffffffffu, mine, (u0 + u) & 31);       // (a result past the end weighs nothing and is zero)
                O.x += v[u].x * f; O.y += v[u].y * f; O.z += v[u].z * f; O.w += v[u].w * f;
            }
        }
    }
    if (sinks) L += exp2f(sinks[head] * LOG2E - (M == -INFINITY ? 0.f : M));
    if (col < VD) {
        const float inv = 1.0f / L;
        *reinterpret_cast<uint2*>(out + (size_t)token * out_stride + (size_t)head * VD + col) = uint2{pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv)};
    }
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

// Rows of an item at most.
WLLM_API int wllm_prefix_attention_rows() { return ROWS; }

// The attention of a planned batch.  pool_pages: pages of the pools; n_tokens: rows of q and out; scratch: nkv * rows * (VD + 2) floats, rows as the plan has them (or the most that a plan of
// this array may have); items_at, tokens_at: their places in the plan; n_items: its items, or -1: its header says; pairs: (item, kv head) pairs, or the most that there may be; ctas: SMs.  sinks, slopes: 32-bit [nq] or null; cap > 0: scores become cap tanh(score / cap).
WLLM_API int wllm_prefix_attention(const void* q, int q_stride, void* out, int out_stride, const void* k_pages, const void* v_pages, long long pool_pages, const int* block_table,
                                   int max_pages, int n_tokens, int nq, int nkv, int page_size, float scale, float cap, const float* sinks, const float* slopes, const int* plan,
                                   int items_at, int tokens_at, int n_items, float* scratch, long long rows, long long pairs, int ctas, int* status, cudaStream_t stream) {
    if (n_tokens <= 0 || pairs <= 0) return WLLM_OK;
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0 || nq / nkv > ROWS || page_size < 16 || (page_size & (page_size - 1)) || pool_pages < 1 || max_pages < 1 || nkv > 65535 || ctas < 1 ||
        !(scale > 0.f) || !(cap >= 0.f) || rows < 1 || items_at < 0 || tokens_at < 0 || pool_pages * nkv > 0x7fffffffLL / page_size ||
        (long long)n_tokens * (q_stride / 8) > 0x7fffffffLL)
        return WLLM_BAD_SIZE;
    if (q_stride % 8 != 0 || out_stride % 4 != 0 || ((uintptr_t)q & 15) || ((uintptr_t)out & 7) || ((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15) || ((uintptr_t)scratch & 15))
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
    return wllm_launch(prefix_merge_kernel, dim3(n_tokens, nkv, (rep * MERGE_BLOCKS + MERGE_WARPS - 1) / MERGE_WARPS), MERGE_WARPS * 32, 0, stream, (bf16*)out, out_stride, plan, rep, rows,
                       (const float*)p.part_o, (const float*)p.part_ml, sinks);
}
