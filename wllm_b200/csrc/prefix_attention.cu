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
// A CTA takes (item, key/value head) pairs blockIdx, + gridDim, ... off the plan's list, so that a captured launch serves plans of any number of items.  Roles by warp:
//   warp 0     brings key and value tiles of 128 keys by TMA through the block table of the item's request, box by box of a page, into a ring of stages;
//   warp 1     one lane issues tcgen05.mma: S = Q K^T (Q and K from shared memory, M 128, N 128) into one of two score buffers, a tile ahead of the softmax, and O += P V (P from
//              tensor memory, over the scores that it came from; V as it lies in the pages, MN-major);
//   warps 2-5  a thread per row: the rows of Q into shared memory, then per tile the scores out of tensor memory, mask, exponentials, running maximum and sum, P back; the row of O is
//              scaled again only when its maximum has grown by more than 2^8.  A warp without rows leaves the tensor core to multiply what lies there: row m of a product
//              depends on row m of its operand alone, and such rows are stored nowhere.
// Tensor memory: O in columns 0 .. 255, the score buffers at 256 and 384.
//
// Head sizes that are no multiple of 64 are widened to one in shared memory: a box copy that reaches past a row's end fills with zeros.  Values of slots behind an item's last key
// (whatever the page holds) are cleared in shared memory before they are multiplied with their weight of zero: 0 x NaN is no zero.
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
constexpr int Q_BYTES = BM * HDP * 2;
constexpr int MOST_STAGES = (227 * 1024 - 1024 - Q_BYTES - BM * 8 - 256) / STAGE;
constexpr int STAGES = MOST_STAGES > 8 ? 8 : MOST_STAGES;
static_assert(STAGES >= 2, "a stage for keys and one for values");
constexpr int SMEM = 1024 + Q_BYTES + STAGES * STAGE + BM * 8 + 256;
constexpr int THREADS = 192;
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
    const int* plan;
    float *part_o, *part_ml;             // [kv heads][rows][VD], [kv heads][rows][2]
    int* status;
};

__global__ void __launch_bounds__(THREADS, 1)
prefix_kernel(const __grid_constant__ Prefix p, const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    extern __shared__ unsigned char smem_raw[];
    pdl_begin();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    const uint32_t q_s = base, ring = q_s + Q_BYTES, rows_s = ring + STAGES * STAGE, bars = rows_s + BM * 8;
    const uint32_t full = bars, empty = full + 8 * STAGES, s_full = empty + 8 * STAGES, q_full = s_full + 16, p_full = q_full + 8, pv_done = p_full + 8, edge_full = pv_done + 8,
                   tmem_slot = edge_full + 8;
    unsigned char* smem = smem_raw + (base - smem_addr(smem_raw));
    struct Row { int src, at; };                             // a row's place in q (in steps of 8 elements), its position
    Row* row_of = reinterpret_cast<Row*>(smem + (rows_s - base));
    volatile uint32_t* tmem_slot_ptr = reinterpret_cast<volatile uint32_t*>(smem + (tmem_slot - base));

    const int n_items = p.plan[PLAN_ITEMS], total = n_items * p.nkv, plan_rows = p.plan[PLAN_ROWS];
    const int* items = p.plan + p.plan[PLAN_AT_ITEMS];
    const int* tokens = p.plan + p.plan[PLAN_AT_TOKENS];
    const int rep = p.nq / p.nkv, page_shift = 31 - __clz(p.page_size);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        mbar_init(s_full, 1); mbar_init(s_full + 8, 1);
        mbar_init(q_full, 4);
        mbar_init(p_full, 4);
        mbar_init(pv_done, 1);
        mbar_init(edge_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tc_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot_ptr;

    if (warp == 0) {
        // ---------------- keys and values ----------------
        const int box_rows = p.page_size < BN ? p.page_size : BN;
        bool ok = true;
        int fill = 0, edges = 0;
        auto load = [&](const int* table, int g, int key0, int key_hi, bool value, int chunk) {
            const int s = fill % STAGES;
            if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * s, ((fill / STAGES) & 1) ^ 1))) { ok = false; return; }
            const int width = value ? VW : KW;
            const uint32_t dst = ring + s * STAGE;
            // a value tile that reaches past the item's last key lands on a barrier of its own, is cleared there, and is announced then
            const bool edge = value && key0 + BN > key_hi;
            const uint32_t bar = edge ? edge_full : full + 8 * s;
            if (lane == 0) mbar_expect_tx(bar, BN * width * 2);
            __syncwarp();
            for (int r0 = lane * box_rows; r0 < BN; r0 += 32 * box_rows) {
                const int key = key0 + r0, index = key >> page_shift;
                int page = index < p.max_pages ? table[index] : 0;
                if (page < 0) page = 0;
                const int row = (page * p.nkv + g) * p.page_size + (key & (p.page_size - 1));
                for (int cb = 0; cb < width / 64; ++cb) tma_load_2d(dst + cb * (BN * 128) + r0 * 128, value ? &v_map : &k_map, bar, chunk * width + cb * 64, row);
            }
            if (edge) {
                if (!__all_sync(0xffffffffu, mbar_wait(edge_full, edges & 1))) { ok = false; return; }
                ++edges;
                const int lo = key_hi - key0;
                for (int i = lane; i < (BN - lo) * (VW / 8); i += 32) {
                    const int row = lo + i / (VW / 8), rest = i % (VW / 8);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(dst + (rest >> 3) * (BN * 128) + row * 128 + (rest & 7) * 16), "r"(0u) : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(full + 8 * s);
            }
            ++fill;
        };
        for (int it = blockIdx.x; it < total && ok; it += gridDim.x) {
            const int* item = items + (it / p.nkv) * PLAN_ITEM;
            const int g = it % p.nkv, lo = item[ITEM_KEY_LO], hi = item[ITEM_KEY_HI], T = (hi - lo + BN - 1) / BN;
            const int* table = p.block_table + (size_t)item[ITEM_REQUEST] * p.max_pages;
            for (int c = 0; c < KC && ok; ++c) load(table, g, lo, hi, false, c);
            for (int n = 0; n < T && ok; ++n) {
                for (int c = 0; c < KC && ok && n + 1 < T; ++c) load(table, g, lo + (n + 1) * BN, hi, false, c);
                for (int c = 0; c < VC && ok; ++c) load(table, g, lo + n * BN, hi, true, c);
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
            int use = 0, tile = 0, done = 0;                     // stages used, tiles begun before this item's, items
            auto scores = [&](int b) -> bool {                   // S = Q K^T of the next tile into buffer b
                for (int c = 0; c < KC; ++c, ++use) {
                    const int s = use % STAGES;
                    if (!mbar_wait(full + 8 * s, (use / STAGES) & 1)) return false;
                    tc_fence_after();
                    const uint32_t kb = ring + s * STAGE;
                    const int steps = min(KW, HD - c * KW + 15) / 16;          // (columns behind the head's are zeros)
                    for (int k = 0; k < steps; ++k) {
                        const int col = c * (KW / 64) + (k >> 2);
                        tc_mma(tmem + S_COL + b * BN, smem_desc(q_s + col * (BM * 128) + (k & 3) * 32), smem_desc(kb + (k >> 2) * (BN * 128) + (k & 3) * 32), IDESC_S, c > 0 || k > 0 ? 1u : 0u);
                    }
                    tc_commit(empty + 8 * s);
                }
                tc_commit(s_full + 8 * b);
                return true;
            };
            for (int it = blockIdx.x; it < total && ok; it += gridDim.x, ++done) {
                const int* item = items + (it / p.nkv) * PLAN_ITEM;
                const int T = (item[ITEM_KEY_HI] - item[ITEM_KEY_LO] + BN - 1) / BN;
                if (!mbar_wait(q_full, done & 1)) { ok = false; break; }
                tc_fence_after();
                ok = scores(tile & 1);
                for (int n = 0; n < T && ok; ++n, ++tile) {
                    if (n + 1 < T && !scores((tile + 1) & 1)) { ok = false; break; }
                    const uint32_t pa = tmem + S_COL + (tile & 1) * BN;
                    for (int c = 0; c < VC && ok; ++c, ++use) {
                        const int s = use % STAGES;
                        if (!mbar_wait(full + 8 * s, (use / STAGES) & 1) || (c == 0 && !mbar_wait(p_full, tile & 1))) { ok = false; break; }
                        tc_fence_after();
                        const uint32_t vb = ring + s * STAGE;
#pragma unroll
                        for (int k = 0; k < BN / 16; ++k)
                            tc_mma_ts(tmem + c * VW, pa + k * 8, smem_desc_mn(vb + k * (16 * 128), BN * 128), IDESC_PV, n > 0 || k > 0 ? 1u : 0u);
                        tc_commit(empty + 8 * s);
                    }
                    if (ok) tc_commit(pv_done);
                }
            }
            if (!ok) atomicExch(p.status, GAVE_UP_MMA);
        }
    } else {
        // ---------------- softmax: a thread per row ----------------
        const int quarter = warp & 3, row = quarter * 32 + lane, tid = threadIdx.x - 64;
        const uint32_t t_lane = tmem + ((uint32_t)(quarter * 32) << 16);
        const float sc = (p.capl > 0.f || p.slopes != nullptr) ? 1.0f : p.scale2;        // capped and biased scores are in powers of two already
        const float pre = p.capl > 0.f ? 1.0f : p.scale2;
        const float cap_in = p.capl > 0.f ? 2.0f * p.scale2 / p.capl : 0.f;
        bool ok = true;
        int tile = 0;
        for (int it = blockIdx.x; it < total; it += gridDim.x) {
            const int* item = items + (it / p.nkv) * PLAN_ITEM;
            const int g = it % p.nkv, lo = item[ITEM_KEY_LO], hi = item[ITEM_KEY_HI], T = (hi - lo + BN - 1) / BN, rows = item[ITEM_TOKENS] * rep;
            const bool own = item[ITEM_OWN] != 0, live = row < rows, warp_live = quarter * 32 < rows;
            {
                Row mine{0, 0};
                if (live) {
                    const int* t = tokens + 2 * (item[ITEM_TOKEN] + row / rep);
                    mine = Row{t[0] * (p.q_stride / 8) + (g * rep + row % rep) * (HD / 8), t[1]};
                }
                row_of[row] = mine;
            }
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (int i = tid; i < rows * (HDP / 8); i += 128) {
                const int r = i / (HDP / 8), chunk = i % (HDP / 8);
                cp_async16(q_s + (chunk >> 3) * (BM * 128) + r * 128 + (((chunk ^ r) & 7) << 4), p.q + (chunk < HD / 8 ? (size_t)(row_of[r].src + chunk) * 8 : 0), chunk < HD / 8);
            }
            asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            const int pos = row_of[row].at;
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            const int last = own ? min(pos, hi - 1) : hi - 1;              // the last key that the row sees
            const float slope2 = (p.slopes != nullptr && live) ? p.slopes[g * rep + row % rep] * LOG2E : 0.f;
            float m_run = -INFINITY, l_run = 0.f;
            for (int n = 0; n < T; ++n, ++tile) {
                const int b = tile & 1, key0 = lo + n * BN;
                if (!__all_sync(0xffffffffu, mbar_wait(s_full + 8 * b, (tile >> 1) & 1))) { ok = false; break; }
                float corr = 1.f;
                bool changed = false;
                if (warp_live) {
                    tc_fence_after();
                    uint32_t sv[4][32];
#pragma unroll
                    for (int h = 0; h < 4; ++h) tc_ld32(t_lane + S_COL + b * BN + 32 * h, sv[h]);
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
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (__all_sync(0xffffffffu, !live || key0 + BN - 1 <= last)) {
#pragma unroll
                        for (int c = 0; c < BN; ++c) mx4[c & 3] = fmaxf(mx4[c & 3], __uint_as_float(sv[c >> 5][c & 31]));
                    } else {
#pragma unroll
                        for (int c = 0; c < BN; ++c) {
                            const float v = key0 + c <= last ? __uint_as_float(sv[c >> 5][c & 31]) : -INFINITY;
                            sv[c >> 5][c & 31] = __float_as_uint(v);
                            mx4[c & 3] = fmaxf(mx4[c & 3], v);
                        }
                    }
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                    const float m_tile = fmaxf(m_run, mx * sc);
                    const float m_new = m_tile > m_run + SLACK ? m_tile : m_run;           // m_run = -inf: takes m_tile
                    const float mbase = m_new == -INFINITY ? 0.f : m_new;
                    corr = fast_exp2(m_run - mbase);
                    float sum4[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t packed[2][32];
#pragma unroll
                    for (int c = 0; c < BN; c += 2) {
                        const float p0 = fast_exp2(fmaf(__uint_as_float(sv[c >> 5][c & 31]), sc, -mbase));
                        const float p1 = fast_exp2(fmaf(__uint_as_float(sv[(c + 1) >> 5][(c + 1) & 31]), sc, -mbase));
                        sum4[(c >> 1) & 3] += p0 + p1;
                        packed[c >> 6][(c >> 1) & 31] = pack_bf16(p0, p1);
                    }
                    l_run = l_run * corr + ((sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
                    changed = live && m_new > m_run;
                    m_run = m_new;
                    tc_st32(t_lane + S_COL + b * BN, packed[0]);
                    tc_st32(t_lane + S_COL + b * BN + 32, packed[1]);
                }
                if (n > 0) {
                    if (!__all_sync(0xffffffffu, mbar_wait(pv_done, (tile - 1) & 1))) { ok = false; break; }        // O of the tile before is complete
                    if (__any_sync(0xffffffffu, changed)) {
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
                }
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full);
            }
            if (ok && !__all_sync(0xffffffffu, mbar_wait(pv_done, (tile - 1) & 1))) ok = false;
            if (ok && warp_live) {
                tc_fence_after();
                const size_t at = (size_t)g * plan_rows + item[ITEM_ROW] + row;
                if (live) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m_run, l_run);
#pragma unroll 1
                for (int c0 = 0; c0 < VD; c0 += 32) {
                    uint32_t ov[32];
                    tc_ld32(t_lane + c0, ov);
                    tc_wait_ld();
                    if (live)
#pragma unroll
                        for (int c = 0; c < 32; c += 4)
                            if (c0 + c < VD)
                                *reinterpret_cast<float4*>(p.part_o + at * VD + c0 + c) = make_float4(__uint_as_float(ov[c]), __uint_as_float(ov[c + 1]), __uint_as_float(ov[c + 2]),
                                                                                                     __uint_as_float(ov[c + 3]));
                }
                tc_fence_before();                       // read before the next item's products are let loose on O (by q_full)
            }
            // every thread of the four warps is done with this item's rows before the next one's are put down; they go on or give up together
            uint32_t all;
            asm volatile("{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %1, 0;\n\tbar.red.and.pred b, 1, 128, a;\n\tselp.u32 %0, 1, 0, b;\n\t}" : "=r"(all) : "r"(ok ? 1u : 0u) : "memory");
            if (!all) {
                if (ok) break;                       // (another warp has recorded why)
                atomicExch(p.status, GAVE_UP_SOFTMAX);
                break;
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

// The merge of a token's results: grid (tokens, kv heads), a warp per (query head, 128 columns)
__global__ void __launch_bounds__(256)
prefix_merge_kernel(bf16* __restrict__ out, int out_stride, const int* __restrict__ plan, int rep, const float* __restrict__ part_o, const float* __restrict__ part_ml,
                    const float* __restrict__ sinks) {
    pdl_begin();
    const int token = blockIdx.x, g = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int* starts = plan + plan[PLAN_AT_STARTS];
    const int first = starts[token], n = starts[token + 1] - first;
    if (n <= 0) return;
    const int* list = plan + plan[PLAN_AT_RESULTS] + first;
    const size_t head0 = (size_t)g * plan[PLAN_ROWS];
    constexpr int BLOCKS = (VD + 127) / 128;
    for (int w = warp; w < rep * BLOCKS; w += 8) {
        const int h = w / BLOCKS, col = (w % BLOCKS) * 128 + lane * 4, head = g * rep + h;
        float M = -INFINITY, L = 0.f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = 0; i0 < n; i0 += 32) {
            const size_t row = i0 + lane < n ? head0 + list[i0 + lane] + h : 0;
            const float2 ml = i0 + lane < n ? *reinterpret_cast<const float2*>(part_ml + row * 2) : make_float2(-INFINITY, 0.f);
            const float M_new = fmaxf(M, warp_max(ml.x)), base = M_new == -INFINITY ? 0.f : M_new;
            const float keep = exp2f(M - base), mine = exp2f(ml.x - base);
            L = L * keep + warp_sum(ml.y * mine);
            O.x *= keep; O.y *= keep; O.z *= keep; O.w *= keep;
            const int count = min(32, n - i0);
            for (int u0 = 0; u0 < count; u0 += 4) {
                float4 v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const size_t at = __shfl_sync(0xffffffffu, row, (u0 + u) & 31);
                    v[u] = u0 + u < count && col < VD ? *reinterpret_cast<const float4*>(part_o + at * VD + col) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float f = __shfl_sync(0xffffffffu, mine, (u0 + u) & 31);
                    if (u0 + u < count) { O.x += v[u].x * f; O.y += v[u].y * f; O.z += v[u].z * f; O.w += v[u].w * f; }
                }
            }
            M = M_new;
        }
        if (sinks) L += exp2f(sinks[head] * LOG2E - (M == -INFINITY ? 0.f : M));
        if (col < VD) {
            const float inv = 1.0f / L;
            uint2 packed{pack_bf16(O.x * inv, O.y * inv), pack_bf16(O.z * inv, O.w * inv)};
            *reinterpret_cast<uint2*>(out + (size_t)token * out_stride + (size_t)head * VD + col) = packed;
        }
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
WLLM_API int wllm_prefix_attention_rows() { return BM; }

// The attention of a planned batch.  pool_pages: pages of the pools; n_tokens: rows of q and out; scratch: nkv * rows * (VD + 2) floats, rows as the plan has them (or the most that a plan of
// this array may have); pairs: (item, kv head) pairs of the plan, or the most that there may be; ctas: SMs.  sinks, slopes: 32-bit [nq] or null; cap > 0: scores become cap tanh(score / cap).
WLLM_API int wllm_prefix_attention(const void* q, int q_stride, void* out, int out_stride, const void* k_pages, const void* v_pages, long long pool_pages, const int* block_table,
                                   int max_pages, int n_tokens, int nq, int nkv, int page_size, float scale, float cap, const float* sinks, const float* slopes, const int* plan,
                                   float* scratch, long long rows, long long pairs, int ctas, int* status, cudaStream_t stream) {
    if (n_tokens <= 0 || pairs <= 0) return WLLM_OK;
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0 || nq / nkv > BM || page_size < 16 || (page_size & (page_size - 1)) || pool_pages < 1 || max_pages < 1 || nkv > 65535 || ctas < 1 ||
        !(scale > 0.f) || !(cap >= 0.f) || rows < 1 || pool_pages * nkv > 0x7fffffffLL / page_size ||
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
    p.scale2 = scale * LOG2E; p.capl = cap * LOG2E; p.slopes = slopes; p.plan = plan; p.status = status;
    p.part_o = scratch; p.part_ml = scratch + (size_t)nkv * rows * VD;
    const int st = wllm_launch(prefix_kernel, dim3((unsigned)(pairs < ctas ? pairs : ctas)), THREADS, SMEM, stream, p, km, vm);
    if (st) return st;
    const int rep = nq / nkv;
    return wllm_launch(prefix_merge_kernel, dim3(n_tokens, nkv), 256, 0, stream, (bf16*)out, out_stride, plan, rep, (const float*)p.part_o, (const float*)p.part_ml, sinks);
}
