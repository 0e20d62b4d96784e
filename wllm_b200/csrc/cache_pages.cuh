// What a call of csrc/cache_pages.cu takes, for it and for its caller (csrc/host_calls.cpp).
#pragma once

// One pool and its moves
struct PagePoolMoves {
    const void* src;
    void* dst;
    long long outer, src_pages, dst_pages, heads, slots, row_bytes, moves;
    const int *src_list, *dst_list, *slot_list;      // slot_list null: whole pages
};
