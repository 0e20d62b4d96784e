// Pages of the cache copied: d_i <- s_i for a list of moves, over every layer of a pool at once, inside a pool or into another one.
//
// A pool is [outer][pages][heads][slots][row] without gaps, `outer` being whatever stands in front of the pages (layers, keys | values).  A move names a page of
// the source pool, one of the destination pool and how many slots of it hold tokens: of every head's run of slots the first `slots` rows are copied, the others stay
// as they are.  A tensor of per-request state is a pool whose pages have one head and one slot.  Several pools may be moved by one launch.
//
// Nothing is computed: the floor is every byte read once and written once at the rate of a plain copy.  The moves travel as kernel parameters (they are known on
// the host, which keeps the block tables), so a launch needs no copy of a list to the device; a launch takes up to MAX_MOVES of them.  A CTA copies a piece of
// one contiguous run (a page of one layer, or one head's slots of it where not all of them are copied) with 16-byte loads, all of a thread's in flight before the
// first is stored.  Moves happen in no order: no destination may be named twice or be a source of the same pool, which the entry point checks.
#include "common.cuh"
#include "cache_pages.cuh"

#include <new>
#include <vector>

constexpr int MAX_POOLS = 16, MAX_MOVES = 512, CP_THREADS = 256, CP_UNROLL = 8;

struct PagePool {
    const unsigned char* src;
    unsigned char* dst;
    long long src_outer, dst_outer;      // bytes between two of `outer`
    int outer, heads, head_bytes, row_bytes;
};
struct PageMove { int pool, src, dst, slots, first; };      // `first`: the move's first CTA
template <int MOVES> struct PageMoves { PagePool pool[MAX_POOLS]; PageMove move[MOVES]; int moves; };

// Units of U bytes (16, or less where rows are no multiple of that); `piece`: units a CTA copies, a multiple of CP_THREADS
template <typename U, int MOVES>
__global__ void __launch_bounds__(CP_THREADS)
copy_pages_kernel(const __grid_constant__ PageMoves<MOVES> p, int piece) {
    pdl_begin();
    int lo = 0, hi = p.moves - 1;
    while (lo < hi) {                    // the last move whose first CTA is not behind this one
        const int mid = (lo + hi + 1) >> 1;
        if (p.move[mid].first <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const PageMove m = p.move[lo];
    const PagePool& q = p.pool[m.pool];
    // a page whose slots are all copied is one run, else every head's slots are
    const long long page = (long long)q.heads * q.head_bytes, part = (long long)m.slots * q.row_bytes;
    const bool whole = part == q.head_bytes;
    const int runs = whole ? 1 : q.heads;
    const long long units = (whole ? page : part) / (int)sizeof(U);
    const int pieces = (int)((units + piece - 1) / piece);
    const int at = (int)blockIdx.x - m.first, k = at % pieces, run = at / pieces % runs, outer = at / pieces / runs;
    const long long inside = (long long)run * q.head_bytes;
    const U* src = reinterpret_cast<const U*>(q.src + outer * q.src_outer + m.src * page + inside);
    U* dst = reinterpret_cast<U*>(q.dst + outer * q.dst_outer + m.dst * page + inside);
    const long long end = min(units, (long long)(k + 1) * piece);
    for (long long i = (long long)k * piece + threadIdx.x; i < end; i += CP_UNROLL * CP_THREADS) {
        U v[CP_UNROLL];
#pragma unroll
        for (int u = 0; u < CP_UNROLL; ++u)
            if (i + u * CP_THREADS < end) v[u] = src[i + u * CP_THREADS];
#pragma unroll
        for (int u = 0; u < CP_UNROLL; ++u)
            if (i + u * CP_THREADS < end) dst[i + u * CP_THREADS] = v[u];
    }
}

enum { PAGES_OUT_OF_RANGE = 7, PAGES_TWICE = 8, POOLS_OVERLAP = 9 };

static bool apart(const void* a, long long na, const void* b, long long nb) {
    return (const char*)a + na <= (const char*)b || (const char*)b + nb <= (const char*)a;
}

template <typename U, int MOVES>
static int launch_pages(const PageMoves<MOVES>& p, int ctas, int piece, cudaStream_t stream) {
    return wllm_launch(copy_pages_kernel<U, MOVES>, dim3(ctas), CP_THREADS, 0, stream, p, piece);
}

// `launched`: kernels launched so far, also when a later one fails
static int copy_pages(const PagePoolMoves* pools, int n, int sms, int* launched, cudaStream_t stream) {
    if (n < 0 || n > MAX_POOLS || sms < 1) return WLLM_BAD_SIZE;
    long long unit = 16, total = 0;
    for (int i = 0; i < n; ++i) {
        const PagePoolMoves& a = pools[i];
        if (a.outer < 1 || a.outer > 0x7fffffff || a.heads < 1 || a.slots < 1 || a.row_bytes < 1 || a.src_pages < 0 || a.dst_pages < 0 || a.moves < 0 ||
            a.heads > 0x7fffffff / (a.slots * a.row_bytes) || a.slots * a.row_bytes > 0x7fffffff)
            return WLLM_BAD_SIZE;
        if (a.moves == 0) continue;
        const long long page = a.heads * a.slots * a.row_bytes;
        while (unit > 1 && (a.row_bytes % unit || (uintptr_t)a.src % unit || (uintptr_t)a.dst % unit)) unit /= 2;
        const long long src_bytes = a.outer * a.src_pages * page, dst_bytes = a.outer * a.dst_pages * page;
        const bool same = a.src == a.dst && a.src_pages == a.dst_pages;
        if (!same && !apart(a.src, src_bytes, a.dst, dst_bytes)) return POOLS_OVERLAP;
        for (int j = 0; j < n; ++j) {
            const PagePoolMoves& b = pools[j];
            if (j == i || b.moves == 0) continue;
            const long long b_page = b.heads * b.slots * b.row_bytes;
            if (!apart(a.dst, dst_bytes, b.dst, b.outer * b.dst_pages * b_page) || !apart(a.dst, dst_bytes, b.src, b.outer * b.src_pages * b_page))
                return POOLS_OVERLAP;
        }
        std::vector<unsigned char> taken((size_t)a.dst_pages, 0);
        for (long long k = 0; k < a.moves; ++k) {
            const int s = a.src_list[k], d = a.dst_list[k], slots = a.slot_list ? a.slot_list[k] : (int)a.slots;
            if (s < 0 || s >= a.src_pages || d < 0 || d >= a.dst_pages || slots < 0 || slots > a.slots) return PAGES_OUT_OF_RANGE;
            if (taken[d]) return PAGES_TWICE;
            taken[d] = 1;
            total += a.outer * a.heads * slots * a.row_bytes;
        }
        if (same)
            for (long long k = 0; k < a.moves; ++k)
                if (taken[a.src_list[k]]) return PAGES_TWICE;
    }
    if (unit < 2) unit = 1;
    // a CTA's piece: 32 KB, less where that would leave SMs without one
    long long piece = CP_THREADS * CP_UNROLL;
    while (piece > CP_THREADS && total / (piece * unit) < 2LL * sms) piece /= 2;
    PageMoves<MAX_MOVES> p;
    long long ctas = 0;
    p.moves = 0;
    auto flush = [&]() -> int {
        if (p.moves == 0) return WLLM_OK;
        int st;
        // few moves: a few hundred bytes of parameters instead of ten thousand
        if (p.moves <= 16) {
            PageMoves<16> few;
            for (int i = 0; i < MAX_POOLS; ++i) few.pool[i] = p.pool[i];
            for (int i = 0; i < p.moves; ++i) few.move[i] = p.move[i];
            few.moves = p.moves;
            st = unit == 16 ? launch_pages<uint4, 16>(few, (int)ctas, (int)piece, stream) : unit >= 4 ? launch_pages<uint32_t, 16>(few, (int)ctas, (int)piece * (int)unit / 4, stream) :
                 unit == 2 ? launch_pages<uint16_t, 16>(few, (int)ctas, (int)piece, stream) : launch_pages<uint8_t, 16>(few, (int)ctas, (int)piece, stream);
        } else {
            st = unit == 16 ? launch_pages<uint4, MAX_MOVES>(p, (int)ctas, (int)piece, stream) : unit >= 4 ? launch_pages<uint32_t, MAX_MOVES>(p, (int)ctas, (int)piece * (int)unit / 4, stream) :
                 unit == 2 ? launch_pages<uint16_t, MAX_MOVES>(p, (int)ctas, (int)piece, stream) : launch_pages<uint8_t, MAX_MOVES>(p, (int)ctas, (int)piece, stream);
        }
        if (st == WLLM_OK) ++*launched;
        p.moves = 0;
        ctas = 0;
        return st;
    };
    for (int i = 0; i < MAX_POOLS; ++i) p.pool[i] = PagePool{};
    for (int i = 0; i < n; ++i) {
        const PagePoolMoves& a = pools[i];
        const long long head = a.slots * a.row_bytes, page = a.heads * head;
        p.pool[i] = PagePool{(const unsigned char*)a.src, (unsigned char*)a.dst, a.src_pages * page, a.dst_pages * page, (int)a.outer, (int)a.heads, (int)head, (int)a.row_bytes};
    }
    for (int i = 0; i < n; ++i) {
        const PagePoolMoves& a = pools[i];
        for (long long k = 0; k < a.moves; ++k) {
            const int slots = a.slot_list ? a.slot_list[k] : (int)a.slots;
            if (slots == 0) continue;
            const bool whole = slots == a.slots;
            const long long run = (whole ? a.heads * a.slots : slots) * a.row_bytes, bytes = piece * unit;
            const long long mine = a.outer * (whole ? 1 : a.heads) * ((run + bytes - 1) / bytes);
            if (mine > 0x7fffffff) return WLLM_BAD_SIZE;
            if (p.moves == MAX_MOVES || ctas + mine > 0x7fffffff) {
                const int st = flush();
                if (st) return st;
            }
            p.move[p.moves++] = PageMove{i, a.src_list[k], a.dst_list[k], slots, (int)ctas};
            ctas += mine;
        }
    }
    return flush();
}

// Every move of every pool; nothing is copied unless all of them are in order.  No exception leaves.
WLLM_API int wllm_copy_pages(const PagePoolMoves* pools, int n, int sms, int* launched, cudaStream_t stream) {
    *launched = 0;
    try {
        return copy_pages(pools, n, sms, launched, stream);
    } catch (const std::bad_alloc&) {
        return WLLM_BAD_SIZE;
    }
}
