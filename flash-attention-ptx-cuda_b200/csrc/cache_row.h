// Where a row of a sequence lies in a KV cache (fa_cache_layout).  Compiles for the host too, where a test walks
// every row of small caches through it, page numbers that name no page among them.
//
// The reference has no cache.
#pragma once

#include "bounded_wait.h"       // FA_HOST_DEVICE

namespace fa {

struct CacheMap {
    const int* block_table;
    int table_stride, page_shift, n_pages;     // page_shift < 0: a block is a sequence
};
// The block of a row (sequence or page; -1: a page number that names none) and the row within it.
struct CacheRow {
    long long block;
    int in_block;
};
FA_HOST_DEVICE CacheRow cache_row(const CacheMap& m, int b, int row) {
    if (m.page_shift < 0) return {(long long)b, row};
    const int page = m.block_table[(long long)b * m.table_stride + (row >> m.page_shift)];
    return {(unsigned)page < (unsigned)m.n_pages ? (long long)page : -1ll, row & ((1 << m.page_shift) - 1)};
}
FA_HOST_DEVICE int sequence_length(const int* seq_lens, int b, int seq_len_kv) {
    if (seq_lens == nullptr) return seq_len_kv;
    const int n = seq_lens[b];
    return n < 0 ? 0 : n < seq_len_kv ? n : seq_len_kv;
}

}  // namespace fa
