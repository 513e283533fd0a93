// C entries of a paged operator's launcher with an error word of the caller's, for the tests. Linked from the library's own object files.
#include "kernels/kernels.h"

using namespace dooms::cuda;

#pragma GCC visibility push(default)
extern "C" int paged_entry_rope_store(void * keys, void * values, const int * table, int n_pages, int page_size, int n_sequences, int max_pages, int n_head_kv, int head_dim,
                                      const float * qkv, int n_head, int n_rows, const int * sequence, const int * at, const int * positions, float * q, int * error) {
    const PagedCache c{keys, values, table, n_pages, page_size, n_sequences, max_pages, n_head_kv, head_dim};
    const RopeSections rope{10000.0, 1, 1, {head_dim / 2, 0, 0, 0}};
    return int(launch_rope_store_paged(c, rope, qkv, (int64_t(n_head) + 2 * n_head_kv) * head_dim, n_head, n_rows, sequence, at, positions, q, false, error, nullptr));
}
#pragma GCC visibility pop
