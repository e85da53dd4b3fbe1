// The paged cache of keys and values (spc3d_cache_append, spc3d_cache_attend): what the host side
// hands to the kernels of cache.hip.  Internal to the library.
#pragma once
#include "attention.h"

namespace spc3d {

// Pages of one cache: keys [page][head][slot][dim], values [page][head][dim][slot], in 8 bits a
// scale for each page and head beside either.  Values lie by element so that a lane of the matrix
// instructions gets its eight tokens of one element with one load.
struct CacheView {
    char *k, *v;
    float *k_scale, *v_scale; // null: not in 8 bits
    uint32_t npages, page, heads, dim;
    int dtype;
};

// Rows starts[b] .. starts[b + 1] of the panels are the newest tokens of sequence b, which holds
// lens[b] with them; its token t lies in page table[b * table_stride + t / page].
struct SeqsView {
    const uint32_t *table, *lens, *starts;
    uint32_t nseq, table_stride, rows, max_rows, max_len;
};

struct AppendArgs {
    CacheView c;
    SeqsView s;
    HeadsView k, v, q, q_out; // q.p null: no queries to rotate
    const float *rotations;   // [position][turned]: cosines, then sines; null: none
    uint32_t turned, q_heads;
    uint32_t each;      // heads of a page that a workgroup takes
    uint32_t rows_each; // rows of queries: 1 or 4
    int dtype; // of the panels
};

struct ReadArgs {
    CacheView c;
    SeqsView s;
    HeadsView q, o;
    float *lse; // [row][head], may be null
    uint32_t heads;
    int32_t window, sinks;
    float scale;
    int dtype;
    uint32_t col_tiles;  // tiles of 16 * columns_per_wave (row, head) pairs of a kv head
    uint32_t splits;     // workgroups that share the tokens of a sequence
    uint32_t share;      // steps of read_step() tokens that each of them has at most
    float *partial;      // [row][head][split][dim + 2], with more than one
};

hipError_t launch_cache_append(const AppendArgs &a, hipStream_t stream);
// (row, head) pairs that a workgroup takes: 16 or 32.
uint32_t read_columns(uint32_t max_rows, uint32_t group);
uint32_t read_step(int cache_dtype);
hipError_t launch_cache_read(const ReadArgs &a, hipStream_t stream);

} // namespace spc3d
