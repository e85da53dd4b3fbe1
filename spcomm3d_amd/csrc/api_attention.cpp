// C ABI: attention over a band (include/spcomm3d_hip.h): argument checks, the band's tiles and
// workspace, the launches of attention.hip.
#include "api_internal.h"
#include "attention.h"

#include <algorithm>
#include <climits>
#include <cmath>

namespace {

// The pieces that spc3d_attend_grad's column kernel works on, for one number of kv heads.
struct KeySchedule {
    uint32_t kv_heads = 0, npieces = 0, nsplits = 0, nslots = 0;
    KeyPiece *pieces = nullptr;
    KeySplit *splits = nullptr;
};

} // namespace

struct spc3d_band {
    uint32_t magic;
    spc3d_ctx *ctx;
    std::vector<uint32_t> rows, cols;
    int32_t window, sinks; // window: INT32_MAX for none
    uint32_t nrows = 0, ncols = 0; // of all sequences
    RowTile *tiles[2] = {nullptr, nullptr}; // of 64 and of 128 rows, the longest walk first
    uint32_t ntiles[2] = {0, 0};
    std::vector<KeySchedule> schedules;
    // spc3d_attend_grad's workspace: sums <dO, o> of every row and head, partial dK and dV.  A
    // block that a call with more heads replaces stays until the band goes: a recorded sequence
    // may use it.
    float *work = nullptr;
    uint64_t work_floats = 0;
    std::vector<void *> retired;
};

namespace {

inline bool live(const spc3d_band *b) { return b && b->magic == kMagicBand && live(b->ctx); }

void free_band(spc3d_band *b)
{
    for (RowTile *t : b->tiles)
        if (t) ctx_free(b->ctx, t);
    for (KeySchedule &s : b->schedules) {
        if (s.pieces) ctx_free(b->ctx, s.pieces);
        if (s.splits) ctx_free(b->ctx, s.splits);
    }
    if (b->work) ctx_free(b->ctx, b->work);
    for (void *p : b->retired)
        ctx_free(b->ctx, p);
    delete b;
}

template <typename T> int to_device(spc3d_ctx *ctx, T **out, const std::vector<T> &host)
{
    if (host.empty())
        return SPC3D_OK;
    const int rc = ctx_alloc(ctx, out, host.size());
    return rc ? rc : copy_h2d(ctx, *out, host.data(), host.size() * sizeof(T));
}

// Columns that the rows at positions pa .. pb see, in steps of kKeyStep: what a tile costs.
int64_t steps_of(int64_t pa, int64_t pb, int64_t ncols, int64_t window, int64_t sinks)
{
    const int64_t end = std::min(pb + 1, ncols), step = kKeyStep;
    if (end <= 0)
        return 0;
    const int64_t lo = std::max<int64_t>(0, pa - window + 1), first = (std::min(sinks, end) + step - 1) / step;
    return first + std::max<int64_t>(0, (end + step - 1) / step - std::max(lo / step, first));
}

std::vector<RowTile> row_tiles(const spc3d_band *b, uint32_t size)
{
    std::vector<std::pair<int64_t, RowTile>> all;
    uint32_t row0 = 0, key0 = 0;
    for (size_t s = 0; s < b->rows.size(); ++s) {
        const uint32_t n = b->rows[s], m = b->cols[s];
        for (uint32_t r = 0; r < n; r += std::min(size, n - r)) {
            RowTile t = {};
            t.row0 = row0 + r;
            t.nrow = std::min(size, n - r);
            t.key0 = key0;
            t.ncols = m;
            t.pos0 = (int32_t)((int64_t)m - n + r);
            all.push_back({steps_of(t.pos0, (int64_t)t.pos0 + t.nrow - 1, m, b->window, b->sinks), t});
        }
        row0 += n;
        key0 += m;
    }
    std::stable_sort(all.begin(), all.end(), [](const auto &x, const auto &y) { return x.first > y.first; });
    std::vector<RowTile> tiles;
    tiles.reserve(all.size());
    for (const auto &p : all)
        tiles.push_back(p.second);
    return tiles;
}

// Tiles of kKeyTile columns, each with the rows that see one of them.  A tile that far more rows
// see than others (the first columns, or any without a window) is cut into pieces of rows, about
// four for each CU over all kv heads and none under 128 rows; the pieces' sums are joined.
void key_pieces(const spc3d_band *b, uint32_t kv_heads, std::vector<KeyPiece> &pieces,
                std::vector<KeySplit> &splits, uint32_t *nslots)
{
    std::vector<KeyPiece> tiles;
    uint64_t total = 0;
    uint32_t row0 = 0, key0 = 0;
    for (size_t s = 0; s < b->rows.size(); ++s) {
        const int64_t n = b->rows[s], m = b->cols[s], off = m - n;
        for (int64_t c = 0; c < m; c += kKeyTile) {
            KeyPiece t = {};
            t.nkey = (uint32_t)std::min<int64_t>(kKeyTile, m - c);
            const int64_t lo = std::max<int64_t>(0, c - off);
            int64_t hi = n;
            if (c >= b->sinks)
                hi = std::min(n, c + t.nkey - 1 + b->window - off);
            t.key0 = key0 + (uint32_t)c;
            t.row0 = row0 + (uint32_t)std::min(lo, n);
            t.nrow = (uint32_t)std::max<int64_t>(0, hi - lo);
            t.pos0 = (int32_t)(lo + off);
            t.col0 = (int32_t)c;
            t.slot = kNoSlot;
            tiles.push_back(t);
            total += t.nrow;
        }
        row0 += (uint32_t)n;
        key0 += (uint32_t)m;
    }
    const uint64_t want = std::max<uint64_t>(1, 4ull * b->ctx->cu_count / kv_heads);
    const uint32_t most = (uint32_t)((std::max<uint64_t>(128, (total + want - 1) / want) + 31) / 32 * 32);
    uint32_t slots = 0;
    for (const KeyPiece &t : tiles) {
        const uint32_t count = (t.nrow + most - 1) / most;
        if (count <= 1) {
            pieces.push_back(t);
            continue;
        }
        const uint32_t each = ((t.nrow + count - 1) / count + 31) / 32 * 32;
        KeySplit sp = {t.key0, t.nkey, slots, 0};
        for (uint32_t r = 0; r < t.nrow; r += each) {
            KeyPiece p = t;
            p.row0 += r;
            p.pos0 += (int32_t)r;
            p.nrow = std::min(each, t.nrow - r);
            p.slot = slots++;
            ++sp.count;
            pieces.push_back(p);
        }
        splits.push_back(sp);
    }
    std::stable_sort(pieces.begin(), pieces.end(),
                     [](const KeyPiece &x, const KeyPiece &y) { return x.nrow > y.nrow; });
    *nslots = slots;
}

int schedule_of(spc3d_band *b, uint32_t kv_heads, KeySchedule **out)
{
    for (KeySchedule &s : b->schedules)
        if (s.kv_heads == kv_heads) {
            *out = &s;
            return SPC3D_OK;
        }
    if (int rc = use_device(b->ctx))
        return rc;
    KeySchedule s;
    s.kv_heads = kv_heads;
    std::vector<KeyPiece> pieces;
    std::vector<KeySplit> splits;
    try {
        key_pieces(b, kv_heads, pieces, splits, &s.nslots);
        b->schedules.reserve(b->schedules.size() + 1);
    } catch (const std::bad_alloc &) {
        return fail(SPC3D_ERR_ALLOC, "host allocation failed");
    }
    s.npieces = (uint32_t)pieces.size();
    s.nsplits = (uint32_t)splits.size();
    int rc = to_device(b->ctx, &s.pieces, pieces);
    if (!rc) rc = to_device(b->ctx, &s.splits, splits);
    if (rc) {
        if (s.pieces) ctx_free(b->ctx, s.pieces);
        if (s.splits) ctx_free(b->ctx, s.splits);
        return rc;
    }
    b->schedules.push_back(s);
    *out = &b->schedules.back();
    return SPC3D_OK;
}

int ensure_work(spc3d_band *b, uint64_t floats)
{
    if (floats <= b->work_floats)
        return SPC3D_OK;
    if (int rc = use_device(b->ctx))
        return rc;
    float *grown = nullptr;
    if (int rc = ctx_alloc(b->ctx, &grown, (size_t)floats))
        return rc;
    if (b->work) {
        try {
            b->retired.push_back(b->work);
        } catch (const std::bad_alloc &) {
            ctx_free(b->ctx, grown);
            return fail(SPC3D_ERR_ALLOC, "host allocation failed");
        }
    }
    b->work = grown;
    b->work_floats = floats;
    return SPC3D_OK;
}

int bad_heads(const char *name, const char *what, int status = SPC3D_ERR_INVALID_ARG)
{
    return fail(status, std::string(name) + ": " + what);
}

// One operand: heads of a panel of at least `rows` rows.
int check_heads(const spc3d_ctx *ctx, const char *name, const spc3d_heads *h, uint64_t rows, int dtype,
                uint32_t dim)
{
    if (!h)
        return bad_heads(name, "NULL");
    if (!live(h->panel))
        return bad_heads(name, "its panel is NULL or destroyed");
    const spc3d_panel *p = h->panel;
    if (p->ctx != ctx)
        return bad_heads(name, "its panel belongs to another context");
    if (h->reserved)
        return bad_heads(name, "reserved word set");
    if (p->dtype != SPC3D_F32 && p->dtype != SPC3D_BF16 && p->dtype != SPC3D_F16)
        return bad_heads(name, "heads are float, bfloat16 or half");
    if (p->dtype != dtype)
        return bad_heads(name, "its type differs from q's", SPC3D_ERR_SIZE_MISMATCH);
    if (!h->heads || !h->dim || h->dim % 8 || h->dim > 128)
        return bad_heads(name, "needs at least one head of 8, 16, .. 128 columns");
    if (h->dim != dim)
        return bad_heads(name, "its heads are not as wide as q's", SPC3D_ERR_SIZE_MISMATCH);
    if ((uint64_t)h->col + (uint64_t)h->heads * h->dim > p->n)
        return bad_heads(name, "its heads end behind the panel's columns", SPC3D_ERR_SIZE_MISMATCH);
    const size_t w = elem_size(p->dtype);
    if (p->n * w % 16 || h->col * w % 16)
        return bad_heads(name, "its rows or its first column are no whole 16-byte vectors");
    if (p->m < rows)
        return bad_heads(name, "its panel has fewer rows than the sequences", SPC3D_ERR_SIZE_MISMATCH);
    return SPC3D_OK;
}

// Whether two operands share memory.  Heads of one panel do when their columns meet.
bool overlap(const spc3d_heads *x, const spc3d_heads *y)
{
    const spc3d_panel *p = x->panel, *q = y->panel;
    if (p->dev == q->dev && p->n == q->n && p->dtype == q->dtype)
        return x->col < y->col + y->heads * y->dim && y->col < x->col + x->heads * x->dim;
    return ranges_overlap(p->dev, panel_bytes(p), q->dev, panel_bytes(q));
}

HeadsView view_of(const spc3d_heads *h)
{
    return HeadsView{(char *)h->panel->dev + h->col * elem_size(h->panel->dtype), h->panel->n};
}

int check_call(const spc3d_ctx *ctx, const spc3d_band *band, const spc3d_heads *q, const spc3d_heads *k,
               const spc3d_heads *v, float scale)
{
    if (!live(ctx))
        return fail(SPC3D_ERR_INVALID_ARG, "context is NULL or destroyed");
    if (!live(band))
        return fail(SPC3D_ERR_INVALID_ARG, "band is NULL or destroyed");
    if (band->ctx != ctx)
        return fail(SPC3D_ERR_INVALID_ARG, "band belongs to another context");
    if (!(scale > 0) || !std::isfinite(scale))
        return fail(SPC3D_ERR_INVALID_ARG, "scale must be positive and finite");
    if (!q || !live(q->panel))
        return fail(SPC3D_ERR_INVALID_ARG, "q is NULL or its panel is destroyed");
    const int dt = q->panel->dtype;
    int rc = check_heads(ctx, "q", q, band->nrows, dt, q->dim);
    if (!rc) rc = check_heads(ctx, "k", k, band->ncols, dt, q->dim);
    if (!rc) rc = check_heads(ctx, "v", v, band->ncols, dt, q->dim);
    if (rc)
        return rc;
    if (k->heads != v->heads || q->heads % k->heads)
        return fail(SPC3D_ERR_SIZE_MISMATCH, "k and v need as many heads as each other, q a multiple of that");
    if ((uint64_t)std::max(band->ntiles[0], 1u) * q->heads > INT_MAX)
        return fail(SPC3D_ERR_TOO_LARGE, "more tiles of rows and heads than a grid holds");
    return SPC3D_OK;
}

int check_lse(const spc3d_ctx *ctx, const spc3d_vals *lse, uint64_t n)
{
    if (!live(lse) || lse->ctx != ctx)
        return fail(SPC3D_ERR_INVALID_ARG, "lse is destroyed or belongs to another context");
    if (lse->dtype != SPC3D_F32 || lse->n < n)
        return fail(SPC3D_ERR_SIZE_MISMATCH, "lse needs a float for every row and head");
    return SPC3D_OK;
}

BandArgs args_of(const spc3d_band *b, const spc3d_heads *q, const spc3d_heads *k, const spc3d_heads *v,
                 float scale, uint32_t *tile_rows)
{
    BandArgs a = {};
    a.q = view_of(q);
    a.k = view_of(k);
    a.v = view_of(v);
    a.heads = q->heads;
    a.kv_heads = k->heads;
    a.dim = q->dim;
    a.window = b->window;
    a.sinks = b->sinks;
    a.scale = scale;
    a.dtype = q->panel->dtype;
    // Tiles of 128 rows read K and V half as often; of 64 rows there are twice as many.  The large
    // ones are taken from two for each CU on.
    const int i = (uint64_t)b->ntiles[1] * q->heads >= 2ull * b->ctx->cu_count;
    *tile_rows = i ? 128 : 64;
    a.tiles = b->tiles[i];
    a.ntiles = b->ntiles[i];
    return a;
}

} // namespace

extern "C" {

int spc3d_band_create(spc3d_ctx *ctx, uint32_t nseq, const uint32_t *rows, const uint32_t *cols,
                      uint32_t window, uint32_t sinks, spc3d_band **out)
{
    if (!out)
        return fail(SPC3D_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (!live(ctx))
        return fail(SPC3D_ERR_INVALID_ARG, "context is NULL or destroyed");
    if (nseq && (!rows || !cols))
        return fail(SPC3D_ERR_INVALID_ARG, "rows or cols is NULL");
    uint64_t nrows = 0, ncols = 0;
    for (uint32_t s = 0; s < nseq; ++s) {
        if (rows[s] > (uint32_t)INT_MAX / 2 || cols[s] > (uint32_t)INT_MAX / 2)
            return fail(SPC3D_ERR_TOO_LARGE, "a sequence of more than 2^30 - 1 rows or columns");
        nrows += rows[s];
        ncols += cols[s];
    }
    if (nrows > UINT32_MAX || ncols > UINT32_MAX)
        return fail(SPC3D_ERR_TOO_LARGE, "more than 2^32 - 1 rows or columns");
    int rc = use_device(ctx);
    if (rc)
        return rc;
    spc3d_band *b = new (std::nothrow) spc3d_band();
    if (!b)
        return fail(SPC3D_ERR_ALLOC, "host allocation failed");
    b->ctx = ctx;
    b->window = window && window < (uint32_t)INT_MAX ? (int32_t)window : INT_MAX;
    b->sinks = window ? (int32_t)std::min(sinks, (uint32_t)INT_MAX / 2) : 0;
    b->nrows = (uint32_t)nrows;
    b->ncols = (uint32_t)ncols;
    try {
        b->rows.assign(rows, rows + nseq);
        b->cols.assign(cols, cols + nseq);
        for (int i = 0; i < 2 && !rc; ++i) {
            const std::vector<RowTile> tiles = row_tiles(b, i ? 128 : 64);
            if (tiles.size() > INT_MAX)
                rc = fail(SPC3D_ERR_TOO_LARGE, "too many tiles of rows");
            b->ntiles[i] = (uint32_t)tiles.size();
            if (!rc) rc = to_device(ctx, &b->tiles[i], tiles);
        }
    } catch (const std::bad_alloc &) {
        rc = fail(SPC3D_ERR_ALLOC, "host allocation failed");
    }
    if (rc) {
        free_band(b);
        return rc;
    }
    b->magic = kMagicBand;
    *out = b;
    return SPC3D_OK;
}

int spc3d_band_destroy(spc3d_band *band)
{
    if (!live(band))
        return fail(SPC3D_ERR_INVALID_ARG, "band is NULL or destroyed");
    if (int rc = refuse_while_capturing(band->ctx))
        return rc;
    (void)hipSetDevice(band->ctx->device);
    band->magic = 0;
    free_band(band); // blocks of the pool: what uses them next is queued behind this band's calls
    return SPC3D_OK;
}

int spc3d_attend(spc3d_ctx *ctx, spc3d_band *band, const spc3d_heads *q, const spc3d_heads *k,
                 const spc3d_heads *v, float scale, const spc3d_heads *o, spc3d_vals *lse)
{
    int rc = check_call(ctx, band, q, k, v, scale);
    if (!rc) rc = check_heads(ctx, "o", o, band->nrows, q->panel->dtype, q->dim);
    if (!rc && lse) rc = check_lse(ctx, lse, (uint64_t)band->nrows * q->heads);
    if (rc)
        return rc;
    if (o->heads != q->heads)
        return fail(SPC3D_ERR_SIZE_MISMATCH, "o needs as many heads as q");
    if (overlap(o, q) || overlap(o, k) || overlap(o, v))
        return fail(SPC3D_ERR_INVALID_ARG, "o overlaps q, k or v");
    rc = use_device(ctx, true);
    if (rc)
        return rc;
    uint32_t tile_rows;
    BandArgs a = args_of(band, q, k, v, scale, &tile_rows);
    a.o = view_of(o);
    a.lse = lse ? (float *)lse->dev : nullptr;
    HIP_TRY(launch_attend(a, tile_rows, ctx->stream));
    return SPC3D_OK;
}

int spc3d_attend_grad(spc3d_ctx *ctx, spc3d_band *band, const spc3d_heads *q, const spc3d_heads *k,
                      const spc3d_heads *v, float scale, const spc3d_heads *o, const spc3d_vals *lse,
                      const spc3d_heads *d_o, const spc3d_heads *dq, const spc3d_heads *dk,
                      const spc3d_heads *dv)
{
    int rc = check_call(ctx, band, q, k, v, scale);
    if (rc)
        return rc;
    const int dt = q->panel->dtype;
    rc = check_heads(ctx, "o", o, band->nrows, dt, q->dim);
    if (!rc) rc = check_heads(ctx, "d_o", d_o, band->nrows, dt, q->dim);
    if (!rc) rc = check_heads(ctx, "dq", dq, band->nrows, dt, q->dim);
    if (!rc) rc = check_heads(ctx, "dk", dk, band->ncols, dt, q->dim);
    if (!rc) rc = check_heads(ctx, "dv", dv, band->ncols, dt, q->dim);
    if (!rc) rc = check_lse(ctx, lse, (uint64_t)band->nrows * q->heads);
    if (rc)
        return rc;
    if (o->heads != q->heads || d_o->heads != q->heads || dq->heads != q->heads || dk->heads != k->heads ||
        dv->heads != k->heads)
        return fail(SPC3D_ERR_SIZE_MISMATCH, "o, d_o and dq need as many heads as q, dk and dv as many as k");
    const spc3d_heads *in[5] = {q, k, v, o, d_o}, *res[3] = {dq, dk, dv};
    for (int i = 0; i < 3; ++i) {
        for (const spc3d_heads *x : in)
            if (overlap(res[i], x))
                return fail(SPC3D_ERR_INVALID_ARG, "a gradient overlaps an input");
        for (int j = 0; j < i; ++j)
            if (overlap(res[i], res[j]))
                return fail(SPC3D_ERR_INVALID_ARG, "two gradients overlap");
    }
    rc = use_device(ctx, true);
    if (rc)
        return rc;
    KeySchedule *s = nullptr;
    rc = schedule_of(band, k->heads, &s);
    if (rc)
        return rc;
    if ((uint64_t)s->npieces * k->heads > INT_MAX || s->nsplits > INT_MAX || k->heads > 65535)
        return fail(SPC3D_ERR_TOO_LARGE, "more tiles of columns and heads than a grid holds");
    const uint64_t deltas = ((uint64_t)band->nrows * q->heads + 3) / 4 * 4;
    rc = ensure_work(band, deltas + partial_floats(s->nslots, k->heads, q->dim));
    if (rc)
        return rc;
    uint32_t tile_rows;
    BandArgs a = args_of(band, q, k, v, scale, &tile_rows);
    a.o = view_of(o);
    a.d_o = view_of(d_o);
    a.dq = view_of(dq);
    a.dk = view_of(dk);
    a.dv = view_of(dv);
    a.lse = (float *)lse->dev;
    a.delta = band->work;
    a.partial = band->work + deltas;
    a.pieces = s->pieces;
    a.splits = s->splits;
    a.npieces = s->npieces;
    a.nsplits = s->nsplits;
    HIP_TRY(launch_attend_dq(a, tile_rows, ctx->stream));
    HIP_TRY(launch_attend_dkv(a, ctx->stream));
    return SPC3D_OK;
}

} // extern "C"
