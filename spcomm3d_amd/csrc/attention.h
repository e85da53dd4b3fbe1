// Attention over a band (spc3d_attend, spc3d_attend_grad): what the host side hands to the
// kernels of attention.hip.  Internal to the library.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace spc3d {

constexpr uint32_t kKeyStep = 64;   // columns that the row kernels take at a time
constexpr uint32_t kKeyTile = 128;  // columns of a task of the column kernel
constexpr uint32_t kNoSlot = 0xffffffffu;

// Heads of a panel: element (t, h, j) at p[t * stride + h * dim + j].
struct HeadsView {
    char *p;         // of the first head's first element
    uint64_t stride; // elements from row to row
};

// A tile of rows: rows row0 .. row0 + nrow of the packed queries, at positions pos0 .. of a
// sequence whose columns are rows key0 .. key0 + ncols of the packed keys.
struct RowTile {
    uint32_t row0, nrow, key0, ncols;
    int32_t pos0;
    uint32_t pad[3];
};

// A piece of a tile of columns: columns col0 .. col0 + nkey of their sequence, rows key0 .. of the
// packed keys.  The rows row0 .. row0 + nrow (from position pos0 on) of every head that shares the
// columns see some of them; in steps of dkv_row_step rows, head after head, this piece takes the steps
// step0 .. step0 + nsteps.
// slot: where its partial sums go, or kNoSlot for the only piece of its tile.
// spread: the tile's first kSpread columns only, by all four wavefronts, each with a quarter of a
// head's elements: the sinks, which every later row sees.
struct KeyPiece {
    uint32_t key0, nkey, row0, nrow;
    int32_t pos0, col0;
    uint32_t step0, nsteps, slot, spread, pad[2];
};
constexpr uint32_t kSpread = 16;
// Whether a wavefront of the column kernel has registers for its values, and the rows of a step,
// for elements of `size` bytes and heads computed as `width` of them.
constexpr bool dkv_keeps_v(uint32_t size, uint32_t width) { return size == 4 || width < 128; }
constexpr uint32_t dkv_row_step(uint32_t size, uint32_t width) { return dkv_keeps_v(size, width) ? 64 : 32; }
// Elements that heads of `dim` are computed as, zeros behind their own.
constexpr uint32_t padded_dim(uint32_t size, uint32_t dim) { return dim <= 64 ? 64 : (dim <= 96 && size == 2 ? 96 : 128); }

// A tile of columns in several pieces: partial sums first .. first + count, then `spread` ones of
// its first columns.
struct KeySplit {
    uint32_t key0, nkey, first, count, spread, pad[3];
};

struct BandArgs {
    HeadsView q, k, v, o, d_o, dq, dk, dv;
    float *lse;   // [row][head]; may be null in the forward call
    // [row][head]: lse in base 2 (+inf for rows that see nothing), then <d_o, o>; nstats each, the
    // last one for rows that are not there
    float *stats;
    uint64_t nstats;
    float *partial;
    const RowTile *tiles;
    const KeyPiece *pieces;
    const KeySplit *splits;
    uint32_t ntiles, npieces, nsplits;
    uint32_t heads, kv_heads, dim;
    int32_t window, sinks; // window: INT32_MAX for none
    float scale;
    int dtype;
};

// Rows of a tile of the forward and the dQ kernel: 64 or 128.
hipError_t launch_attend(const BandArgs &a, uint32_t tile_rows, hipStream_t stream);
hipError_t launch_attend_dq(const BandArgs &a, uint32_t tile_rows, hipStream_t stream);
hipError_t launch_attend_dkv(const BandArgs &a, hipStream_t stream);
// Panels of the types that only these calls take.
hipError_t launch_fill_short(int dtype, void *p, uint64_t n, float value, hipStream_t stream);
uint64_t partial_floats(uint32_t nslots, uint32_t kv_heads, uint32_t dim);

} // namespace spc3d
