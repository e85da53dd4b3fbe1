// C ABI: attention over a band (include/spcomm3d_hip.h): argument checks, the band's tiles and
// workspace, the launches of attention.hip.
#include "api_internal.h"
#include "attention.h"
#include "cache.h"

#include <algorithm>
#include <climits>
#include <cmath>
#include <functional>

namespace {

// The pieces that spc3d_attend_grad's column kernel works on, for one number and kind of heads.
struct KeySchedule {
    uint32_t kv_heads = 0, group = 0, row_step = 0, npieces = 0, nsplits = 0, nslots = 0;
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
    // spc3d_attend_grad's workspace: lse and <dO, o> of every row and head, partial dK and dV.  A
    // block that a call with more heads replaces stays until the band goes: a recorded sequence
    // may use it.
    float *work = nullptr;
    uint64_t work_floats = 0;
    std::vector<void *> retired;
};

struct spc3d_cache {
    uint32_t magic;
    spc3d_ctx *ctx;
    CacheView view;
    bool owned = true; // false: the caller's device memory (spc3d_cache_wrap)
    float *work = nullptr; // sums of the workgroups that share a sequence, see spc3d_band
    uint64_t work_floats = 0;
    std::vector<void *> retired;
};

namespace {

inline bool live(const spc3d_cache *c) { return c && c->magic == kMagicCache && live(c->ctx); }
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

// How many units of work the longest of `slots` workers gets when each in turn takes the next of
// `costs` (descending).
uint64_t makespan(const std::vector<uint64_t> &costs, size_t slots)
{
    if (costs.size() <= slots)
        return costs.empty() ? 0 : costs.front();
    std::vector<uint64_t> heap(slots, 0); // the least loaded on top
    for (uint64_t c : costs) {
        std::pop_heap(heap.begin(), heap.end(), std::greater<uint64_t>());
        heap.back() += c;
        std::push_heap(heap.begin(), heap.end(), std::greater<uint64_t>());
    }
    return *std::max_element(heap.begin(), heap.end());
}

// Tiles of kKeyTile columns, each with the rows that see one of them, cut into pieces of steps
// where that ends sooner.  Rows that see a tile for its sinks alone are pieces of their own.
// The choice goes by what the parts of a call cost on an MI355X, in steps (64 rows, 6 us with
// two workgroups on a CU, heads of 128 in 16 bits): half a step to begin and end a piece, two more
// to write its partial sums, half a step of the whole GPU for the launch that joins them and 1/512
// for each piece in it.
void key_pieces(const spc3d_band *b, uint32_t kv_heads, uint32_t group, uint32_t row_step, std::vector<KeyPiece> &pieces,
                std::vector<KeySplit> &splits, uint32_t *nslots)
{
    std::vector<KeyPiece> tiles;
    uint32_t row0 = 0, key0 = 0;
    uint64_t longest = 1;
    auto add = [&](KeyPiece t, int64_t lo, int64_t hi, int64_t off) { // rows lo .. hi of the sequence
        t.row0 = row0 + (uint32_t)lo;
        t.nrow = (uint32_t)std::max<int64_t>(0, hi - lo);
        t.pos0 = (int32_t)(lo + off);
        t.nsteps = (t.nrow + row_step - 1) / row_step * group;
        t.slot = kNoSlot;
        longest = std::max<uint64_t>(longest, t.nsteps);
        tiles.push_back(t);
    };
    for (size_t s = 0; s < b->rows.size(); ++s) {
        const int64_t n = b->rows[s], m = b->cols[s], off = m - n;
        for (int64_t c = 0; c < m; c += kKeyTile) {
            KeyPiece t = {};
            t.nkey = (uint32_t)std::min<int64_t>(kKeyTile, m - c);
            t.key0 = key0 + (uint32_t)c;
            t.col0 = (int32_t)c;
            const int64_t lo = std::min(n, std::max<int64_t>(0, c - off));
            const int64_t near = std::min(n, std::max(lo, c + t.nkey - 1 + b->window - off)); // the window's rows
            const bool spread = c < b->sinks && b->sinks - c <= (int64_t)kSpread && near < n;
            add(t, lo, c < b->sinks && !spread ? n : near, off);
            if (spread) {
                t.spread = 1;
                add(t, near, n, off);
            }
        }
        row0 += (uint32_t)n;
        key0 += (uint32_t)m;
    }
    // the longest piece allowed, by trial
    const size_t slots = std::max<size_t>(1, 2 * (size_t)b->ctx->cu_count / kv_heads);
    auto count_of = [&](const KeyPiece &t, uint64_t most) {
        const uint64_t all = t.spread ? (t.nsteps * 5ull + 7) / 8 : t.nsteps; // a step of the sinks costs five eighths
        return (uint32_t)std::max<uint64_t>(1, (all + most - 1) / most);
    };
    uint64_t best = longest, best_cost = UINT64_MAX;
    std::vector<uint64_t> costs;
    for (uint64_t most = longest, before = 0; most >= 1; most = most * 3 / 4) {
        if (most == before)
            break;
        before = most;
        costs.clear();
        uint64_t joined = 0;
        for (size_t i = 0; i < tiles.size(); ++i) {
            const KeyPiece &t = tiles[i];
            const uint32_t count = count_of(t, most);
            const bool split = count > 1 || t.spread || (i + 1 < tiles.size() && tiles[i + 1].spread);
            const uint64_t each = 512ull * t.nsteps * row_step / 64 * (t.spread ? 5 : 8) / 8 / count;
            for (uint32_t k = 0; k < count; ++k)
                costs.push_back(each + 256 + (split ? 1024 : 0));
            joined += split ? count : 0;
        }
        if (costs.size() > 16 * slots && best_cost != UINT64_MAX)
            break;
        std::sort(costs.begin(), costs.end(), std::greater<uint64_t>());
        const uint64_t cost = makespan(costs, slots) + (joined ? 256 + joined * kv_heads : 0);
        if (cost < best_cost) {
            best_cost = cost;
            best = most;
        }
    }
    uint32_t next = 0;
    std::vector<std::pair<uint64_t, KeyPiece>> all;
    for (size_t i = 0; i < tiles.size(); ++i) {
        const KeyPiece &t = tiles[i];
        const uint32_t count = count_of(t, best);
        const bool lone = count == 1 && !t.spread && !(i + 1 < tiles.size() && tiles[i + 1].spread);
        if (!lone && !t.spread)
            splits.push_back(KeySplit{t.key0, t.nkey, next, count, 0, {}});
        if (t.spread)
            splits.back().spread = count;
        for (uint32_t k = 0; k < count; ++k) {
            KeyPiece p = t;
            p.step0 = (uint32_t)((uint64_t)t.nsteps * k / count);
            p.nsteps = (uint32_t)((uint64_t)t.nsteps * (k + 1) / count) - p.step0;
            if (!lone)
                p.slot = next++;
            all.push_back({t.spread ? p.nsteps * 5ull / 8 : p.nsteps, p});
        }
    }
    std::stable_sort(all.begin(), all.end(), [](const auto &x, const auto &y) { return x.first > y.first; });
    for (const auto &p : all)
        pieces.push_back(p.second);
    *nslots = next;
}

int schedule_of(spc3d_band *b, uint32_t kv_heads, uint32_t group, uint32_t row_step, KeySchedule **out)
{
    for (KeySchedule &s : b->schedules)
        if (s.kv_heads == kv_heads && s.group == group && s.row_step == row_step) {
            *out = &s;
            return SPC3D_OK;
        }
    if (int rc = use_device(b->ctx))
        return rc;
    KeySchedule s;
    s.kv_heads = kv_heads;
    s.group = group;
    s.row_step = row_step;
    std::vector<KeyPiece> pieces;
    std::vector<KeySplit> splits;
    try {
        key_pieces(b, kv_heads, group, row_step, pieces, splits, &s.nslots);
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

// The workspace of a band or a cache with room for so many floats.
template <typename H> int ensure_work(H *b, uint64_t floats)
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
    if (p->n > 1u << 22)
        return bad_heads(name, "its panel has more than 2^22 columns", SPC3D_ERR_TOO_LARGE);
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
    // ones are taken from two for each CU on, for small heads from 11 / 4 on (causal, 64 / 128 rows, us;
    // heads of 128: 256 tiles 89 / 107, 512 70 / 69, 640 92 / 79, 1024 213 / 170; heads of 64: 512
    // 38 / 45, 640 51 / 56, 704 66 / 62, 800 80 / 71).
    const uint64_t large = (uint64_t)b->ntiles[1] * q->heads;
    const int i = 4 * large >= (q->dim > 64 ? 8ull : 11ull) * b->ctx->cu_count;
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
    rc = schedule_of(band, k->heads, q->heads / k->heads,
                     dkv_row_step((uint32_t)elem_size(dt), padded_dim((uint32_t)elem_size(dt), q->dim)), &s);
    if (rc)
        return rc;
    if ((uint64_t)s->npieces * k->heads > INT_MAX || s->nsplits > INT_MAX || k->heads > 65535)
        return fail(SPC3D_ERR_TOO_LARGE, "more tiles of columns and heads than a grid holds");
    const uint64_t stats = ((uint64_t)band->nrows * q->heads + 1 + 3) / 4 * 4;
    rc = ensure_work(band, 2 * stats + partial_floats(s->nslots, k->heads, q->dim));
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
    a.stats = band->work;
    a.nstats = stats;
    a.partial = band->work + 2 * stats;
    a.pieces = s->pieces;
    a.splits = s->splits;
    a.npieces = s->npieces;
    a.nsplits = s->nsplits;
    HIP_TRY(launch_attend_dq(a, tile_rows, ctx->stream));
    HIP_TRY(launch_attend_dkv(a, ctx->stream));
    return SPC3D_OK;
}

/* ---- the paged cache ------------------------------------------------------ */

namespace {

int make_cache(spc3d_ctx *ctx, int dtype, uint32_t npages, uint32_t page, uint32_t heads, uint32_t dim,
               void *const *mem, spc3d_cache **out)
{
    if (!out)
        return fail(SPC3D_ERR_INVALID_ARG, "out is NULL");
    *out = nullptr;
    if (!live(ctx))
        return fail(SPC3D_ERR_INVALID_ARG, "context is NULL or destroyed");
    if (dtype != SPC3D_BF16 && dtype != SPC3D_F16 && dtype != SPC3D_F8)
        return fail(SPC3D_ERR_INVALID_ARG, "a cache holds bfloat16, half or 8 bits");
    if (page != 16 && page != 32 && page != 64 && page != 128)
        return fail(SPC3D_ERR_INVALID_ARG, "pages have 16, 32, 64 or 128 tokens");
    if (!heads || !dim || dim > 128 || dim % (dtype == SPC3D_F8 ? 16 : 8))
        return fail(SPC3D_ERR_INVALID_ARG, "a cache needs heads of 8, 16, .. 128 elements (8 bits: 16, 32, ..)");
    if (heads > 65535 || npages == UINT32_MAX)
        return fail(SPC3D_ERR_TOO_LARGE, "more than 65535 heads or 2^32 - 2 pages");
    int rc = use_device(ctx);
    if (rc)
        return rc;
    const uint64_t units = (uint64_t)npages * heads;
    const bool f8 = dtype == SPC3D_F8;
    const size_t bytes[4] = {(size_t)units * page * dim * elem_size(dtype), (size_t)units * page * dim * elem_size(dtype),
                             f8 ? (size_t)units * 4 : 0, f8 ? (size_t)units * 4 : 0};
    void *at[4] = {nullptr, nullptr, nullptr, nullptr};
    if (mem) {
        for (int i = 0; i < 4 && !rc; ++i) {
            if (i >= 2 && !f8 && mem[i])
                return fail(SPC3D_ERR_INVALID_ARG, "scales belong to a cache in 8 bits");
            rc = check_wrapped(ctx, mem[i], bytes[i]);
            for (int j = 0; j < i && !rc; ++j)
                if (bytes[i] && ranges_overlap(mem[i], bytes[i], mem[j], bytes[j]))
                    rc = fail(SPC3D_ERR_INVALID_ARG, "keys, values and scales overlap");
            at[i] = bytes[i] ? mem[i] : nullptr;
        }
        if (rc)
            return rc;
    }
    spc3d_cache *c = new (std::nothrow) spc3d_cache();
    if (!c)
        return fail(SPC3D_ERR_ALLOC, "host allocation failed");
    c->ctx = ctx;
    c->owned = !mem;
    for (int i = 0; i < 4 && !mem && !rc; ++i)
        rc = dev_alloc_bytes(ctx, &at[i], bytes[i]);
    if (rc) {
        for (void *p : at)
            if (p) (void)hipFree(p);
        delete c;
        return rc;
    }
    c->view = CacheView{(char *)at[0], (char *)at[1], (float *)at[2], (float *)at[3], npages, page, heads, dim, dtype};
    c->magic = kMagicCache;
    *out = c;
    return SPC3D_OK;
}

int check_seqs(const spc3d_cache_seqs *s)
{
    if (!s)
        return fail(SPC3D_ERR_INVALID_ARG, "seqs is NULL");
    if (s->reserved)
        return fail(SPC3D_ERR_INVALID_ARG, "reserved word of spc3d_cache_seqs set");
    if (s->nseq && s->rows && (!s->table || !s->lens || !s->starts))
        return fail(SPC3D_ERR_INVALID_ARG, "table, lens or starts is NULL");
    for (const void *p : {s->table, s->lens, s->starts})
        if (reinterpret_cast<uintptr_t>(p) % 4)
            return fail(SPC3D_ERR_INVALID_ARG, "table, lens or starts is not 4-byte aligned");
    if (s->max_len > (uint32_t)INT_MAX / 2 || s->max_rows > (uint32_t)INT_MAX / 2)
        return fail(SPC3D_ERR_TOO_LARGE, "a sequence of more than 2^30 - 1 tokens or rows");
    return SPC3D_OK;
}

SeqsView view_of(const spc3d_cache_seqs *s)
{
    return SeqsView{(const uint32_t *)s->table, (const uint32_t *)s->lens, (const uint32_t *)s->starts, s->nseq,
                    s->table_stride, s->rows, std::min(s->max_rows, s->rows), s->max_len};
}

// What either call over a cache checks of itself and of the operand `h`.
int check_cached(const spc3d_ctx *ctx, const spc3d_cache *cache, const spc3d_cache_seqs *seqs, const char *name,
                 const spc3d_heads *h)
{
    if (!live(ctx))
        return fail(SPC3D_ERR_INVALID_ARG, "context is NULL or destroyed");
    if (!live(cache))
        return fail(SPC3D_ERR_INVALID_ARG, "cache is NULL or destroyed");
    if (cache->ctx != ctx)
        return fail(SPC3D_ERR_INVALID_ARG, "cache belongs to another context");
    if (int rc = check_seqs(seqs))
        return rc;
    if (!h || !live(h->panel))
        return bad_heads(name, "NULL, or its panel is destroyed");
    const int dt = h->panel->dtype;
    if (dt != SPC3D_BF16 && dt != SPC3D_F16)
        return bad_heads(name, "operands of a cache are bfloat16 or half");
    if (cache->view.dtype != SPC3D_F8 && cache->view.dtype != dt)
        return bad_heads(name, "its type is not the cache's", SPC3D_ERR_SIZE_MISMATCH);
    return check_heads(ctx, name, h, seqs->rows, dt, cache->view.dim);
}

bool in_cache(const spc3d_cache *c, const spc3d_heads *h)
{
    const size_t units = (size_t)c->view.npages * c->view.heads;
    const size_t bytes = units * c->view.page * c->view.dim * elem_size(c->view.dtype);
    const void *const p = h->panel->dev;
    const size_t n = panel_bytes(h->panel);
    return ranges_overlap(p, n, c->view.k, bytes) || ranges_overlap(p, n, c->view.v, bytes) ||
           (c->view.k_scale && (ranges_overlap(p, n, c->view.k_scale, 4 * units) ||
                                ranges_overlap(p, n, c->view.v_scale, 4 * units)));
}

} // namespace

int spc3d_cache_create(spc3d_ctx *ctx, int dtype, uint32_t npages, uint32_t page, uint32_t heads, uint32_t dim,
                       spc3d_cache **out)
{
    return make_cache(ctx, dtype, npages, page, heads, dim, nullptr, out);
}

int spc3d_cache_wrap(spc3d_ctx *ctx, int dtype, uint32_t npages, uint32_t page, uint32_t heads, uint32_t dim, void *k,
                     void *v, void *k_scale, void *v_scale, spc3d_cache **out)
{
    void *const mem[4] = {k, v, k_scale, v_scale};
    return make_cache(ctx, dtype, npages, page, heads, dim, mem, out);
}

int spc3d_cache_destroy(spc3d_cache *c)
{
    if (!live(c))
        return fail(SPC3D_ERR_INVALID_ARG, "cache is NULL or destroyed");
    if (int rc = refuse_while_capturing(c->ctx))
        return rc;
    (void)hipSetDevice(c->ctx->device);
    (void)hipStreamSynchronize(c->ctx->stream);
    if (c->owned)
        for (void *p : {(void *)c->view.k, (void *)c->view.v, (void *)c->view.k_scale, (void *)c->view.v_scale})
            if (p) (void)hipFree(p);
    if (c->work) ctx_free(c->ctx, c->work);
    for (void *p : c->retired)
        ctx_free(c->ctx, p);
    c->magic = 0;
    delete c;
    return SPC3D_OK;
}

int spc3d_cache_device_ptrs(spc3d_cache *c, void **k, void **v, void **k_scale, void **v_scale)
{
    if (!live(c))
        return fail(SPC3D_ERR_INVALID_ARG, "cache is NULL or destroyed");
    if (k) *k = c->view.k;
    if (v) *v = c->view.v;
    if (k_scale) *k_scale = c->view.k_scale;
    if (v_scale) *v_scale = c->view.v_scale;
    return SPC3D_OK;
}

int spc3d_cache_append(spc3d_ctx *ctx, spc3d_cache *cache, const spc3d_cache_seqs *seqs, const spc3d_heads *k,
                       const spc3d_heads *v, const spc3d_panel *rotations, const spc3d_heads *q,
                       const spc3d_heads *q_out)
{
    int rc = check_cached(ctx, cache, seqs, "k", k);
    if (rc)
        return rc;
    const int dt = k->panel->dtype;
    const uint32_t dim = cache->view.dim;
    rc = check_heads(ctx, "v", v, seqs->rows, dt, dim);
    if (rc)
        return rc;
    if (k->heads != cache->view.heads || v->heads != cache->view.heads)
        return fail(SPC3D_ERR_SIZE_MISMATCH, "k and v need as many heads as the cache");
    if (!q != !q_out)
        return fail(SPC3D_ERR_INVALID_ARG, "q and q_out come together");
    if (q) {
        rc = check_heads(ctx, "q", q, seqs->rows, dt, dim);
        if (!rc) rc = check_heads(ctx, "q_out", q_out, seqs->rows, dt, dim);
        if (rc)
            return rc;
        if (q->heads != q_out->heads)
            return fail(SPC3D_ERR_SIZE_MISMATCH, "q_out needs as many heads as q");
        if (overlap(q_out, q) || overlap(q_out, k) || overlap(q_out, v))
            return fail(SPC3D_ERR_INVALID_ARG, "q_out overlaps q, k or v");
        if (in_cache(cache, q_out))
            return fail(SPC3D_ERR_INVALID_ARG, "q_out overlaps the cache");
    }
    if (in_cache(cache, k) || in_cache(cache, v) || (q && in_cache(cache, q)))
        return fail(SPC3D_ERR_INVALID_ARG, "an operand overlaps the cache");
    if (rotations) {
        if (!live(rotations) || rotations->ctx != ctx)
            return fail(SPC3D_ERR_INVALID_ARG, "rotations is destroyed or belongs to another context");
        if (rotations->dtype != SPC3D_F32 || rotations->m < seqs->max_len || rotations->n > dim)
            return fail(SPC3D_ERR_SIZE_MISMATCH,
                        "rotations needs a row of floats for every position, no longer than a head");
        if (rotations->n % 16)
            return fail(SPC3D_ERR_INVALID_ARG, "a multiple of 16 elements of a head is rotated");
        if (q_out && ranges_overlap(rotations->dev, panel_bytes(rotations), q_out->panel->dev, panel_bytes(q_out->panel)))
            return fail(SPC3D_ERR_INVALID_ARG, "q_out overlaps rotations");
    }
    AppendArgs a = {};
    a.c = cache->view;
    a.s = view_of(seqs);
    const uint64_t pages = (uint64_t)seqs->nseq * ((a.s.max_rows + a.c.page - 2) / a.c.page + 1) * a.c.heads * 2;
    if (pages + seqs->rows > INT_MAX)
        return fail(SPC3D_ERR_TOO_LARGE, "more pages and rows than a grid holds");
    rc = use_device(ctx, true);
    if (rc)
        return rc;
    a.k = view_of(k);
    a.v = view_of(v);
    if (q) {
        a.q = view_of(q);
        a.q_out = view_of(q_out);
        a.q_heads = q->heads;
    }
    if (rotations && rotations->n) {
        a.rotations = (const float *)rotations->dev;
        a.turned = rotations->n;
    }
    a.dtype = dt;
    // A head of a page for each workgroup while there are few, four where that still leaves eight
    // workgroups a CU: what they look up before they begin is then a smaller part.
    a.each = pages / 4 >= 8ull * ctx->cu_count ? 4 : 1;
    a.rows_each = seqs->rows / 4 >= 8ull * ctx->cu_count ? 4 : 1;
    HIP_TRY(launch_cache_append(a, ctx->stream));
    return SPC3D_OK;
}

int spc3d_cache_attend(spc3d_ctx *ctx, spc3d_cache *cache, const spc3d_cache_seqs *seqs, const spc3d_heads *q,
                       float scale, uint32_t window, uint32_t sinks, const spc3d_heads *o, spc3d_vals *lse)
{
    int rc = check_cached(ctx, cache, seqs, "q", q);
    if (rc)
        return rc;
    if (!(scale > 0) || !std::isfinite(scale))
        return fail(SPC3D_ERR_INVALID_ARG, "scale must be positive and finite");
    rc = check_heads(ctx, "o", o, seqs->rows, q->panel->dtype, cache->view.dim);
    if (!rc && lse) rc = check_lse(ctx, lse, (uint64_t)seqs->rows * q->heads);
    if (rc)
        return rc;
    if (q->heads % cache->view.heads || o->heads != q->heads)
        return fail(SPC3D_ERR_SIZE_MISMATCH, "q needs a multiple of the cache's heads, o as many as q");
    if (overlap(o, q) || in_cache(cache, o))
        return fail(SPC3D_ERR_INVALID_ARG, "o overlaps q or the cache");
    ReadArgs a = {};
    a.c = cache->view;
    a.s = view_of(seqs);
    a.q = view_of(q);
    a.o = view_of(o);
    a.lse = lse ? (float *)lse->dev : nullptr;
    a.heads = q->heads;
    a.window = window && window < (uint32_t)INT_MAX ? (int32_t)window : INT_MAX;
    a.sinks = window ? (int32_t)std::min(sinks, (uint32_t)INT_MAX / 2) : 0;
    a.scale = scale;
    a.dtype = q->panel->dtype;
    const uint32_t group = q->heads / a.c.heads, cols = read_columns(a.s.max_rows, group);
    const uint64_t tiles = ((uint64_t)a.s.max_rows * group + cols - 1) / cols;
    const uint64_t groups = (uint64_t)seqs->nseq * tiles * a.c.heads;
    // Shares of a sequence's steps: such that the longest sequences would make eight workgroups for each
    // CU (of sequences of several lengths most are shorter, and a share that has no tokens ends at
    // once), but at least a step for each of a workgroup's four wavefronts; none for few steps, which
    // end sooner than a second launch would (700 tokens, 22 steps of 32: 7.6 us, in shares 10.0).
    const uint64_t step = read_step(a.c.dtype);
    uint64_t steps = ((uint64_t)seqs->max_len + step - 1) / step;
    if (a.window != INT_MAX)
        steps = std::min(steps, ((uint64_t)window + a.s.max_rows + step - 1) / step + 1 + ((uint64_t)a.sinks + step - 1) / step);
    const uint64_t share = groups * steps / (8ull * ctx->cu_count);
    a.share = (uint32_t)(steps <= 24 ? 24 : std::max<uint64_t>(4, (share + 3) / 4 * 4));
    a.splits = (uint32_t)std::max<uint64_t>(1, (steps + a.share - 1) / a.share);
    a.col_tiles = (uint32_t)tiles;
    if (groups * a.splits > INT_MAX || (uint64_t)seqs->rows * q->heads / 8 > INT_MAX)
        return fail(SPC3D_ERR_TOO_LARGE, "more rows and heads than a grid holds");
    rc = use_device(ctx, true);
    if (rc)
        return rc;
    if (a.splits > 1) {
        rc = ensure_work(cache, (uint64_t)seqs->rows * q->heads * a.splits * (a.c.dim + 4));
        if (rc)
            return rc;
        a.partial = cache->work;
    }
    HIP_TRY(launch_cache_read(a, ctx->stream));
    return SPC3D_OK;
}

} // extern "C"
