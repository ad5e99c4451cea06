// lm_api.hip -- the C entries of the language-model operators (rotary
// positions, the paged cache and its attention): checks of arguments before
// any device work, then one launch or two.
#include <cmath>
#include <initializer_list>
#include <new>
#include <utility>

#include "mfft_internal.hpp"

using mfft::fail;
using mfft::hip_fail;

namespace {

constexpr int kMaxPairs = 256;
constexpr int64_t kMaxPositions = (int64_t)1 << 24;

struct Extent {
    const char* lo;
    const char* hi;
};

// Byte range of a strided array (strides >= 0, in elements; sizes >= 1).
Extent extent(const void* p, std::initializer_list<int64_t> sizes, const int64_t* strides, int64_t last, int elem) {
    int64_t top = last;
    int i = 0;
    for (int64_t n : sizes) top += (n - 1) * strides[i++];
    return {(const char*)p, (const char*)p + top * elem};
}
bool overlap(const Extent& a, const Extent& b) { return a.lo < b.hi && b.lo < a.hi; }

// Whether the elements of a strided output are distinct: each dimension, from
// the smallest stride up, steps past everything below it.
bool distinct(std::initializer_list<int64_t> sizes, const int64_t* strides, int64_t last) {
    int64_t n[4], s[4];
    int k = 0;
    for (int64_t v : sizes) {
        n[k] = v;
        s[k] = strides[k];
        ++k;
    }
    for (int i = 0; i < k; ++i)
        for (int j = i + 1; j < k; ++j)
            if (s[j] < s[i]) {
                std::swap(s[i], s[j]);
                std::swap(n[i], n[j]);
            }
    int64_t reach = last;
    for (int i = 0; i < k; ++i) {
        if (n[i] == 1) continue;
        if (s[i] < reach) return false;
        reach += (n[i] - 1) * s[i];
    }
    return true;
}

int dtype_size(int dtype) { return dtype == MFFT_F32 ? 4 : 2; }

int check_dtype(int dtype, bool f32) {
    if (dtype == MFFT_F16 || dtype == MFFT_BF16 || (f32 && dtype == MFFT_F32)) return MFFT_OK;
    return fail(MFFT_ERR_TYPE, "unsupported element type %d", dtype);
}

constexpr int64_t kMaxStride = (int64_t)1 << 40;  // elements

// Strides not negative, and the whole array within 2^42 elements, so that no
// offset comes near 64 bits.
int check_strides(const char* what, std::initializer_list<int64_t> sizes, const int64_t* s) {
    int i = 0;
    for (int64_t n : sizes) {
        if (s[i] < 0 || s[i] > kMaxStride || (n > 1 && s[i] > ((int64_t)1 << 42) / (n - 1)))
            return fail(MFFT_ERR_VALUE, "%s: stride %lld is negative or too large", what, (long long)s[i]);
        ++i;
    }
    return MFFT_OK;
}

bool aligned(const void* p, int n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) == 0; }

int check_cache(const mfft_cache* c) {
    if (!c) return fail(MFFT_ERR_VALUE, "cache must not be NULL");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(MFFT_ERR_VALUE, "cache buffers must not be NULL");
    if (!mfft::attend_supported(c->head_dim))
        return fail(MFFT_ERR_UNSUPPORTED, "head_dim must be 64, 96, 128 or 256, got %d", c->head_dim);
    if (c->page_size < 16 || c->page_size > 1024 || c->page_size % 16)
        return fail(MFFT_ERR_VALUE, "page_size must be a multiple of 16 in [16, 1024], got %d", c->page_size);
    if (c->kv_heads < 1 || c->kv_heads > 4096) return fail(MFFT_ERR_VALUE, "kv_heads must be in [1, 4096], got %d", c->kv_heads);
    if (c->pages < 1 || c->pages > 0x7fffffff) return fail(MFFT_ERR_VALUE, "pages must be in [1, 2^31), got %lld", (long long)c->pages);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return fail(MFFT_ERR_VALUE, "cache codes must be 16-byte aligned and scales 4-byte aligned");
    return MFFT_OK;
}

int check_sequences(int64_t tokens, int32_t sequences, int32_t width, int64_t stride, const int32_t* table,
                    const int32_t* lengths, const char* what) {
    if (tokens < 0 || tokens > 0x7fffffff) return fail(MFFT_ERR_VALUE, "tokens must be in [0, 2^31), got %lld", (long long)tokens);
    if (sequences < 1) return fail(MFFT_ERR_VALUE, "sequences must be >= 1, got %d", sequences);
    if (width < 1 || stride < 0 || stride > kMaxStride)
        return fail(MFFT_ERR_VALUE, "page_table must have at least one column, got %d (stride %lld)", width, (long long)stride);
    if (!table || !lengths) return fail(MFFT_ERR_VALUE, "page_table and %s must not be NULL", what);
    if (!aligned(table, 4) || !aligned(lengths, 4)) return fail(MFFT_ERR_VALUE, "page_table and %s must be 4-byte aligned", what);
    return MFFT_OK;
}

int check_device(const mfft_rotary* r) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
    if (r && r->device != dev)
        return fail(MFFT_ERR_RUNTIME, "rotary plan was created on device %d but device %d is current", r->device, dev);
    return MFFT_OK;
}

}  // namespace

extern "C" {

// axis_of: NULL with one axis
static int create_rotary(mfft_rotary** out, const double* frequencies, const int32_t* axis_of, int32_t pairs, int32_t axes,
                         int64_t max_positions, double amplitude, int layout) {
    mfft::clear_error();
    if (!out) return fail(MFFT_ERR_VALUE, "out must not be NULL");
    *out = nullptr;
    if (!frequencies) return fail(MFFT_ERR_VALUE, "frequencies must not be NULL");
    if (pairs < 1 || pairs > kMaxPairs) return fail(MFFT_ERR_VALUE, "pairs must be in [1, %d], got %d", kMaxPairs, pairs);
    if (max_positions < 1 || max_positions > kMaxPositions)
        return fail(MFFT_ERR_VALUE, "max_positions must be in [1, 2^24], got %lld", (long long)max_positions);
    if (layout != MFFT_ROTARY_HALF && layout != MFFT_ROTARY_INTERLEAVED)
        return fail(MFFT_ERR_VALUE, "unknown rotary layout %d", layout);
    if (!std::isfinite(amplitude)) return fail(MFFT_ERR_VALUE, "amplitude must be finite");
    for (int j = 0; j < pairs; ++j)
        if (!std::isfinite(frequencies[j]) || std::fabs(frequencies[j]) > 1e3)
            return fail(MFFT_ERR_VALUE, "frequency %d must be finite and at most 1000 radians a position", j);
    for (int j = 0; axis_of && j < pairs; ++j)
        if (axis_of[j] < 0 || axis_of[j] >= axes)
            return fail(MFFT_ERR_VALUE, "axis_of[%d] must be in [0, %d), got %d", j, axes, axis_of[j]);
    mfft_rotary* r = nullptr;
    try {
        r = new mfft_rotary();
        const int64_t lo_rows = (int64_t)1 << mfft::kRotaryLoLog2;
        const int64_t hi_rows = (max_positions + lo_rows - 1) / lo_rows;
        auto rows = [&](int64_t count, int64_t step, long double m) {
            std::vector<float2> w((size_t)(count * pairs));
            for (int64_t p = 0; p < count; ++p)
                for (int j = 0; j < pairs; ++j) {
                    const long double x = (long double)(p * step) * (long double)frequencies[j];
                    w[(size_t)(p * pairs + j)] = make_float2((float)(m * cosl(x)), (float)(m * sinl(x)));
                }
            return w;
        };
        const std::vector<float2> lo = rows(lo_rows < max_positions ? lo_rows : max_positions, 1, 1.0L);
        const std::vector<float2> hi = rows(hi_rows, lo_rows, (long double)amplitude);
        std::vector<float2> axis((pairs + 7) / 8);
        for (int j = 0; axis_of && j < pairs; ++j) ((uint8_t*)axis.data())[j] = (uint8_t)axis_of[j];
        hipStream_t us = nullptr;
        int rc = MFFT_OK;
        hipError_t e = hipGetDevice(&r->device);
        if (e != hipSuccess) rc = hip_fail(e, "hipGetDevice");
        if (rc == MFFT_OK) rc = mfft::upload_stream(r->device, &us);
        if (rc == MFFT_OK) rc = mfft::upload(&r->lo, lo, &r->table_bytes, us);
        if (rc == MFFT_OK) rc = mfft::upload(&r->hi, hi, &r->table_bytes, us);
        if (rc == MFFT_OK) rc = mfft::upload(&r->axis, axis, &r->table_bytes, us);
        if (us) {
            e = hipStreamSynchronize(us);  // also after a failure: the host tables die here
            if (e != hipSuccess && rc == MFFT_OK) rc = hip_fail(e, "hipStreamSynchronize(rotary tables)");
        }
        if (rc != MFFT_OK) {
            mfft_rotary_destroy(r);
            return rc;
        }
        r->t = {r->lo, r->hi, max_positions, pairs, layout, axes, (const uint8_t*)r->axis};
        *out = r;
        return MFFT_OK;
    } catch (const std::bad_alloc&) {
        mfft_rotary_destroy(r);
        return fail(MFFT_ERR_RUNTIME, "out of host memory for the rotary tables");
    } catch (...) {
        mfft_rotary_destroy(r);
        return fail(MFFT_ERR_RUNTIME, "internal error while building the rotary tables");
    }
}

int mfft_rotary_create(mfft_rotary** out, const double* frequencies, int32_t pairs, int64_t max_positions,
                       double amplitude, int layout) {
    return create_rotary(out, frequencies, nullptr, pairs, 1, max_positions, amplitude, layout);
}

int mfft_rotary_create_axes(mfft_rotary** out, const double* frequencies, const int32_t* axis_of, int32_t pairs,
                            int32_t axes, int64_t max_positions, double amplitude, int layout) {
    mfft::clear_error();
    if (out) *out = nullptr;
    if (axes < 1 || axes > MFFT_MAX_AXES) return fail(MFFT_ERR_VALUE, "axes must be in [1, %d], got %d", MFFT_MAX_AXES, axes);
    if (!axis_of) return fail(MFFT_ERR_VALUE, "axis_of must not be NULL");
    return create_rotary(out, frequencies, axis_of, pairs, axes, max_positions, amplitude, layout);
}

int mfft_rotary_destroy(mfft_rotary* r) {
    if (!r) return MFFT_OK;
    if (r->axis) (void)hipFree(r->axis);
    if (r->lo) (void)hipFree(r->lo);
    if (r->hi) (void)hipFree(r->hi);
    delete r;
    return MFFT_OK;
}

static int execute_rotary(const mfft_rotary* r, const mfft_rotary_args* a, int64_t axis_stride, void* stream) {
    if (int rc = check_dtype(a->dtype, true)) return rc;
    if (a->direction != MFFT_FORWARD && a->direction != MFFT_INVERSE)
        return fail(MFFT_ERR_VALUE, "unsupported direction %d", a->direction);
    if (a->batch < 0 || a->tokens < 0 || a->heads < 0 || a->batch > 0x7fffffff || a->tokens > 0x7fffffff)
        return fail(MFFT_ERR_VALUE, "batch, tokens and heads must be in [0, 2^31)");
    if (a->head_dim < 2 * r->t.pairs || a->head_dim % 2 || a->head_dim > 65536)
        return fail(MFFT_ERR_VALUE, "head_dim must be even, at least the %d rotated channels and at most 65536, got %d",
                    2 * r->t.pairs, a->head_dim);
    if (int rc = check_strides("in", {a->batch, a->tokens, (int64_t)a->heads}, a->in_strides)) return rc;
    if (int rc = check_strides("out", {a->batch, a->tokens, (int64_t)a->heads}, a->out_strides)) return rc;
    if (int rc = check_strides("positions", {a->batch, a->tokens}, a->position_strides)) return rc;
    if (int rc = check_device(r)) return rc;
    if (a->batch == 0 || a->tokens == 0 || a->heads == 0) return MFFT_OK;
    if (!a->in || !a->out || !a->positions) return fail(MFFT_ERR_VALUE, "in, out and positions must not be NULL");
    const int es = dtype_size(a->dtype);
    if (!aligned(a->in, es) || !aligned(a->out, es) || !aligned(a->positions, a->positions_64 ? 8 : 4))
        return fail(MFFT_ERR_VALUE, "in, out and positions must be aligned to their elements");
    if (!distinct({a->batch, a->tokens, a->heads}, a->out_strides, a->head_dim))
        return fail(MFFT_ERR_VALUE, "out's strides make its elements overlap");
    const bool same = a->in == a->out && a->in_strides[0] == a->out_strides[0] &&
                      a->in_strides[1] == a->out_strides[1] && a->in_strides[2] == a->out_strides[2];
    if (!same && overlap(extent(a->in, {a->batch, a->tokens, (int64_t)a->heads}, a->in_strides, a->head_dim, es),
                         extent(a->out, {a->batch, a->tokens, (int64_t)a->heads}, a->out_strides, a->head_dim, es)))
        return fail(MFFT_ERR_VALUE, "in and out must not overlap (except as the same tensor)");
    if (!mfft::rotary_launch_fits(r->t, *a))
        return fail(MFFT_ERR_UNSUPPORTED, "batch=%lld of %lld tokens needs a launch of 2^32 work-items or more; split it",
                    (long long)a->batch, (long long)a->tokens);
    const hipError_t e = mfft::launch_rotary(r->t, *a, axis_stride, (hipStream_t)stream);
    return e == hipSuccess ? MFFT_OK : hip_fail(e, "kernel launch");
}

int mfft_rotary_execute(const mfft_rotary* r, const mfft_rotary_args* a, void* stream) {
    mfft::clear_error();
    if (!r || !a) return fail(MFFT_ERR_VALUE, "rotary and args must not be NULL");
    if (r->t.axes > 1) return fail(MFFT_ERR_VALUE, "the rotary takes positions of %d axes: mfft_rotary_execute_axes", r->t.axes);
    return execute_rotary(r, a, 0, stream);
}

int mfft_rotary_execute_axes(const mfft_rotary* r, const mfft_rotary_args* a, int64_t axis_stride, void* stream) {
    mfft::clear_error();
    if (!r || !a) return fail(MFFT_ERR_VALUE, "rotary and args must not be NULL");
    if (int rc = check_strides("positions", {(int64_t)r->t.axes}, &axis_stride)) return rc;
    return execute_rotary(r, a, axis_stride, stream);
}

static int append(const mfft_cache* c, const mfft_rotary* r, const mfft_append_args* a, const mfft::Positions& at, void* stream) {
    if (int rc = check_cache(c)) return rc;
    if (!a) return fail(MFFT_ERR_VALUE, "args must not be NULL");
    if (int rc = check_dtype(a->dtype, true)) return rc;
    if (int rc = check_sequences(a->tokens, a->sequences, a->table_width, a->table_stride, a->page_table, a->starts, "starts"))
        return rc;
    if (!a->offsets && a->tokens != a->sequences)
        return fail(MFFT_ERR_VALUE, "without offsets each sequence takes one token: %lld tokens, %d sequences",
                    (long long)a->tokens, a->sequences);
    if (a->offsets && !aligned(a->offsets, 4)) return fail(MFFT_ERR_VALUE, "offsets must be 4-byte aligned");
    if (r && 2 * r->t.pairs > c->head_dim)
        return fail(MFFT_ERR_VALUE, "the rotary turns %d channels of a head, the cache's heads have %d", 2 * r->t.pairs, c->head_dim);
    if (int rc = check_strides("k", {a->tokens, (int64_t)c->kv_heads}, a->k_strides)) return rc;
    if (int rc = check_strides("v", {a->tokens, (int64_t)c->kv_heads}, a->v_strides)) return rc;
    if (a->q) {
        if (a->q_heads < 1 || a->q_heads > 65536) return fail(MFFT_ERR_VALUE, "q_heads must be in [1, 65536], got %d", a->q_heads);
        if (int rc = check_strides("q", {a->tokens, (int64_t)a->q_heads}, a->q_strides)) return rc;
        if (int rc = check_strides("q_out", {a->tokens, (int64_t)a->q_heads}, a->q_out_strides)) return rc;
    }
    if (int rc = check_device(r)) return rc;
    if (a->tokens == 0) return MFFT_OK;
    const int es = dtype_size(a->dtype);
    if (!a->k || !a->v || !aligned(a->k, es) || !aligned(a->v, es))
        return fail(MFFT_ERR_VALUE, "k and v must not be NULL and be aligned to their elements");
    if (a->q) {
        if (!a->q_out || !aligned(a->q, es) || !aligned(a->q_out, es))
            return fail(MFFT_ERR_VALUE, "q_out must not be NULL, and q and q_out aligned to their elements");
        if (!distinct({a->tokens, (int64_t)a->q_heads}, a->q_out_strides, c->head_dim))
            return fail(MFFT_ERR_VALUE, "q_out's strides make its elements overlap");
        const bool same = a->q == a->q_out && a->q_strides[0] == a->q_out_strides[0] && a->q_strides[1] == a->q_out_strides[1];
        const Extent qo = extent(a->q_out, {a->tokens, (int64_t)a->q_heads}, a->q_out_strides, c->head_dim, es);
        if (!same && overlap(extent(a->q, {a->tokens, (int64_t)a->q_heads}, a->q_strides, c->head_dim, es), qo))
            return fail(MFFT_ERR_VALUE, "q and q_out must not overlap (except as the same tensor)");
    }
    if (!mfft::append_launch_fits(r ? r->t : mfft::RotaryTables{}, *c, *a))
        return fail(MFFT_ERR_UNSUPPORTED, "%lld tokens need a launch of 2^32 work-items or more; split the call", (long long)a->tokens);
    const hipError_t e = mfft::launch_append(r ? r->t : mfft::RotaryTables{}, *c, *a, at, (hipStream_t)stream);
    return e == hipSuccess ? MFFT_OK : hip_fail(e, "kernel launch");
}

int mfft_cache_append(const mfft_cache* c, const mfft_rotary* r, const mfft_append_args* a, void* stream) {
    mfft::clear_error();
    if (r && r->t.axes > 1)
        return fail(MFFT_ERR_VALUE, "the rotary takes positions of %d axes: mfft_cache_append_at", r->t.axes);
    return append(c, r, a, mfft::Positions{}, stream);
}

int mfft_cache_append_at(const mfft_cache* c, const mfft_rotary* r, const mfft_append_args* a, const void* positions,
                         int64_t axis_stride, int64_t token_stride, int32_t positions_64, void* stream) {
    mfft::clear_error();
    if (!r || !a) return fail(MFFT_ERR_VALUE, "rotary and args must not be NULL");
    if (int rc = check_strides("positions", {(int64_t)r->t.axes}, &axis_stride)) return rc;
    if (a->tokens > 0) {
        if (int rc = check_strides("positions", {a->tokens}, &token_stride)) return rc;
        if (!positions || !aligned(positions, positions_64 ? 8 : 4))
            return fail(MFFT_ERR_VALUE, "positions must not be NULL and be aligned to their elements");
    }
    return append(c, r, a, mfft::Positions{positions, axis_stride, token_stride, positions_64}, stream);
}

int mfft_cache_read(const mfft_cache* c, const mfft_read_args* a, void* stream) {
    mfft::clear_error();
    if (int rc = check_cache(c)) return rc;
    if (!a) return fail(MFFT_ERR_VALUE, "args must not be NULL");
    if (int rc = check_dtype(a->dtype, true)) return rc;
    if (int rc = check_sequences(a->tokens, a->sequences, a->table_width, a->table_stride, a->page_table, a->starts, "starts"))
        return rc;
    if (a->offsets && !aligned(a->offsets, 4)) return fail(MFFT_ERR_VALUE, "offsets must be 4-byte aligned");
    if (!a->offsets && a->tokens % a->sequences)
        return fail(MFFT_ERR_VALUE, "without offsets every sequence has as many rows: %lld tokens, %d sequences",
                    (long long)a->tokens, a->sequences);
    if (int rc = check_strides("k", {a->tokens, (int64_t)c->kv_heads}, a->k_strides)) return rc;
    if (int rc = check_strides("v", {a->tokens, (int64_t)c->kv_heads}, a->v_strides)) return rc;
    if (a->tokens == 0) return MFFT_OK;
    const int es = dtype_size(a->dtype);
    // (the stride of one token, or of one head, is not used)
    auto keeps = [&](const int64_t* st) { return (a->tokens == 1 || st[0] * es % 16 == 0) && (c->kv_heads == 1 || st[1] * es % 16 == 0); };
    if (!a->k || !a->v || !aligned(a->k, 16) || !aligned(a->v, 16) || !keeps(a->k_strides) || !keeps(a->v_strides))
        return fail(MFFT_ERR_VALUE, "k and v must not be NULL, and 16-byte aligned with strides that keep it so");
    if (!distinct({a->tokens, (int64_t)c->kv_heads}, a->k_strides, c->head_dim) ||
        !distinct({a->tokens, (int64_t)c->kv_heads}, a->v_strides, c->head_dim))
        return fail(MFFT_ERR_VALUE, "k's or v's strides make its elements overlap");
    const Extent ek = extent(a->k, {a->tokens, (int64_t)c->kv_heads}, a->k_strides, c->head_dim, es);
    const Extent ev = extent(a->v, {a->tokens, (int64_t)c->kv_heads}, a->v_strides, c->head_dim, es);
    if (overlap(ek, ev)) return fail(MFFT_ERR_VALUE, "k and v must not overlap");
    const int64_t codes = c->pages * c->kv_heads * (int64_t)c->page_size * c->head_dim;
    for (const Extent& e : {ek, ev})
        for (const void* p : {c->k, c->v})
            if (overlap(e, Extent{(const char*)p, (const char*)p + codes}))
                return fail(MFFT_ERR_VALUE, "k and v must not overlap the cache");
    if (!mfft::read_launch_fits(*c, *a))
        return fail(MFFT_ERR_UNSUPPORTED, "%lld tokens need a launch of 2^32 work-items or more; split the call", (long long)a->tokens);
    const hipError_t e = mfft::launch_read(*c, *a, (hipStream_t)stream);
    return e == hipSuccess ? MFFT_OK : hip_fail(e, "kernel launch");
}

static int check_attend(const mfft_cache* c, const mfft_attend_args* a) {
    if (int rc = check_cache(c)) return rc;
    if (!a) return fail(MFFT_ERR_VALUE, "args must not be NULL");
    if (int rc = check_dtype(a->dtype, false)) return rc;
    if (int rc = check_sequences(a->tokens, a->sequences, a->table_width, a->table_stride, a->page_table, a->lengths, "lengths"))
        return rc;
    if (a->offsets && !aligned(a->offsets, 4)) return fail(MFFT_ERR_VALUE, "offsets must be 4-byte aligned");
    if (!a->offsets && a->tokens % a->sequences)
        return fail(MFFT_ERR_VALUE, "without offsets every sequence has as many queries: %lld tokens, %d sequences",
                    (long long)a->tokens, a->sequences);
    if (a->q_heads < 1 || a->q_heads % c->kv_heads || a->q_heads > 65536)
        return fail(MFFT_ERR_VALUE, "q_heads must be a multiple of the cache's %d heads, at most 65536, got %d", c->kv_heads, a->q_heads);
    if (a->tokens > ((int64_t)1 << 30) / a->q_heads)
        return fail(MFFT_ERR_UNSUPPORTED, "more than 2^30 query rows (%lld tokens of %d heads); split the call",
                    (long long)a->tokens, a->q_heads);
    if (!std::isfinite(a->scale) || a->scale < 0.0f) return fail(MFFT_ERR_VALUE, "scale must be finite and not negative");
    if (a->window < 0 || a->window > (int64_t)1 << 30) return fail(MFFT_ERR_VALUE, "window must be in [0, 2^30]");
    if ((int64_t)a->table_width * c->page_size > (int64_t)1 << 30)
        return fail(MFFT_ERR_VALUE, "page_table holds more than 2^30 positions a sequence");
    if (a->max_length < 0) return fail(MFFT_ERR_VALUE, "max_length must not be negative");
    if (int rc = check_strides("q", {a->tokens, (int64_t)a->q_heads}, a->q_strides)) return rc;
    if (int rc = check_strides("out", {a->tokens, (int64_t)a->q_heads}, a->out_strides)) return rc;
    return MFFT_OK;
}

static int check_options(const mfft_attend_options* o) {
    if (!o) return fail(MFFT_ERR_VALUE, "options must not be NULL");
    if (o->sinks < 0 || o->sinks > (int64_t)1 << 30) return fail(MFFT_ERR_VALUE, "sinks must be in [0, 2^30]");
    if (o->prefix_pages) {
        if (o->groups < 1 || (!o->prefix_groups && o->groups != 1))
            return fail(MFFT_ERR_VALUE, "prefix_pages must be of one group at least, and of one only without prefix_groups, got %d",
                        o->groups);
        if (!aligned(o->prefix_pages, 4) || !aligned(o->prefix_groups, 4))
            return fail(MFFT_ERR_VALUE, "prefix_pages and prefix_groups must be 4-byte aligned");
    } else if (o->prefix_groups) {
        return fail(MFFT_ERR_VALUE, "prefix_groups say whose prefix_pages are: give prefix_pages");
    }
    return MFFT_OK;
}

static int workspace(const mfft_cache* c, const mfft_attend_args* a, const mfft_attend_options& o, int64_t* bytes) {
    if (!bytes) return fail(MFFT_ERR_VALUE, "bytes must not be NULL");
    *bytes = 0;
    if (int rc = check_attend(c, a)) return rc;
    *bytes = a->tokens ? mfft::attend_workspace(*c, *a, o) : 0;
    return MFFT_OK;
}

static int attend(const mfft_cache* c, const mfft_attend_args* a, const mfft_attend_options& opt, void* stream) {
    if (int rc = check_attend(c, a)) return rc;
    if (a->tokens == 0) return MFFT_OK;
    const int64_t D = c->head_dim;
    // (the stride of one token, or of one head, is not used)
    const int64_t n[2] = {a->tokens, a->q_heads};
    auto keeps = [&](const int64_t* s, int m) { return (n[0] == 1 || s[0] % m == 0) && (n[1] == 1 || s[1] % m == 0); };
    if (!a->q || !a->out || !aligned(a->q, 16) || !aligned(a->out, 8) || !keeps(a->q_strides, 8) || !keeps(a->out_strides, 4))
        return fail(MFFT_ERR_VALUE, "q must be 16-byte and out 8-byte aligned, with strides that keep it so");
    if (a->lse && !aligned(a->lse, 4)) return fail(MFFT_ERR_VALUE, "lse must be 4-byte aligned");
    if (!distinct({a->tokens, (int64_t)a->q_heads}, a->out_strides, D))
        return fail(MFFT_ERR_VALUE, "out's strides make its elements overlap");
    const Extent o = extent(a->out, {a->tokens, (int64_t)a->q_heads}, a->out_strides, D, 2);
    if (overlap(extent(a->q, {a->tokens, (int64_t)a->q_heads}, a->q_strides, D, 2), o))
        return fail(MFFT_ERR_VALUE, "q and out must not overlap");
    if (!mfft::attend_launch_fits(*c, *a, opt))
        return fail(MFFT_ERR_UNSUPPORTED, "%lld tokens need a launch of 2^32 work-items or more; split the call", (long long)a->tokens);
    const int64_t need = mfft::attend_workspace(*c, *a, opt);
    if (need > 0) {
        if (!a->workspace || a->workspace_bytes < need)
            return fail(MFFT_ERR_VALUE, "the call needs %lld bytes of workspace, got %lld", (long long)need,
                        (long long)(a->workspace ? a->workspace_bytes : 0));
        if (!aligned(a->workspace, 256)) return fail(MFFT_ERR_VALUE, "workspace must be 256-byte aligned");
    }
    const hipError_t e = mfft::launch_attend(*c, *a, opt, (hipStream_t)stream);
    return e == hipSuccess ? MFFT_OK : hip_fail(e, "kernel launch");
}

int mfft_cache_attend_workspace(const mfft_cache* c, const mfft_attend_args* a, int64_t* bytes) {
    mfft::clear_error();
    return workspace(c, a, mfft_attend_options{}, bytes);
}

int mfft_cache_attend_with_workspace(const mfft_cache* c, const mfft_attend_args* a, const mfft_attend_options* o,
                                     int64_t* bytes) {
    mfft::clear_error();
    if (int rc = check_options(o)) return rc;
    return workspace(c, a, *o, bytes);
}

int mfft_cache_attend(const mfft_cache* c, const mfft_attend_args* a, void* stream) {
    mfft::clear_error();
    return attend(c, a, mfft_attend_options{}, stream);
}

int mfft_cache_attend_with(const mfft_cache* c, const mfft_attend_args* a, const mfft_attend_options* o, void* stream) {
    mfft::clear_error();
    if (int rc = check_options(o)) return rc;
    return attend(c, a, *o, stream);
}

}  // extern "C"
