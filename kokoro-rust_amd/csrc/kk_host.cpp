// kk_host.cpp -- host-only rules of the C ABI: durations_from_logits and the ragged layout tables
// (the bit-exact integer contract of the path), and the checks of an ids-level item and of the cache
// operators' arguments.  Plain C++, built into the library and, for the sanitizer tests, on its own.
#include "kk_host.h"

#include <cmath>

namespace kk {

std::string ids_item_error(const kk_item& it, int b) {
    const std::string sb = std::to_string(b);
    if (it.ids == nullptr || it.ref_s == nullptr) return "item " + sb + ": null input";
    if (it.n_ids < 2 || it.n_ids > 512) return "item " + sb + ": input_ids length outside [2, 512]";
    if (!(std::isfinite(it.speed) && it.speed > 0.f)) return "item " + sb + ": speed must be positive and finite";
    for (int i = 0; i < it.n_ids; i++)  // the message is built only for a failing id
        if (it.ids[i] < 0 || it.ids[i] >= 178)
            return "item " + sb + ": token id " + std::to_string(it.ids[i]) + " out of range";
    if (it.noise_kind != KK_NOISE_COUNTER && it.noise_kind != KK_NOISE_FIXED) return "item " + sb + ": unknown noise kind";
    return "";
}

// Sizes that keep every index of the kernels in its type: row and token numbers (and a window added to them) in 32 bits, a
// launch's blocks times their threads below 2^32.
constexpr int64_t kMostRows = (int64_t)1 << 28, kMostTokens = (int64_t)1 << 30, kMostSeqs = (int64_t)1 << 20;
constexpr int kMostHeads = 4096;

static bool aligned(const void* p, size_t to) { return (uintptr_t)p % to == 0; }
static size_t value_bytes(int type) { return type == KK_F32 ? 4 : 2; }

std::string norm_rope_error(const kk_norm_rope* a) {
    if (!a) return "null arguments";
    if (a->type != KK_BF16 && a->type != KK_F16 && a->type != KK_F32) return "unknown type " + std::to_string(a->type);
    if (a->dim < 2 || a->dim > 512 || a->dim % 2) return "head dimension " + std::to_string(a->dim) + " is not even and in [2, 512]";
    if (a->rows < 0 || a->rows > kMostRows) return "rows out of range";
    if (a->q_heads < 0 || a->k_heads < 0 || a->q_heads > kMostHeads || a->k_heads > kMostHeads) return "head count out of range";
    if (a->rot < 0 || a->rot > a->dim || a->rot % 2) return "rot " + std::to_string(a->rot) + " is not even and in [0, dim]";
    if (a->norm != 0 && a->norm != 1) return "norm is 0 or 1";
    if (a->norm && !(a->eps >= 0.f && std::isfinite(a->eps))) return "eps must be at least 0 and finite";
    if (a->interleaved != 0 && a->interleaved != 1) return "interleaved is 0 or 1";
    if (a->rot && !a->freq && !(a->theta > 0 && std::isfinite(a->theta))) return "theta must be positive and finite";
    if (a->rows == 0 || a->q_heads + a->k_heads == 0) return "";
    if ((a->q_heads && (!a->q || !a->q_out)) || (a->k_heads && (!a->k || !a->k_out)) || !a->pos) return "null array";
    const size_t e = value_bytes(a->type);
    if (!aligned(a->q, e) || !aligned(a->k, e) || !aligned(a->q_out, e) || !aligned(a->k_out, e) || !aligned(a->pos, 4) ||
        !aligned(a->q_weight, 4) || !aligned(a->k_weight, 4) || !aligned(a->freq, 8))
        return "an array is not aligned to its values";
    auto strides = [](const void* in, const void* out, int64_t row, int64_t head, int64_t out_row, int64_t out_head) {
        return in != out || (row == out_row && head == out_head);
    };
    if ((a->q_heads && !strides(a->q, a->q_out, a->q_row, a->q_head, a->q_out_row, a->q_out_head)) ||
        (a->k_heads && !strides(a->k, a->k_out, a->k_row, a->k_head, a->k_out_row, a->k_out_head)))
        return "an output in place of its input has other strides";
    return "";
}

std::string kv_batch_error(const kk_kv_cache* c, const kk_kv_batch* b) {
    if (!c || !b) return "null arguments";
    if (c->type != KK_KV_INT8 && c->type != KK_KV_E4M3) return "unknown cache type " + std::to_string(c->type);
    if (c->dim != 64 && c->dim != 96 && c->dim != 128 && c->dim != 192 && c->dim != 256)
        return "head dimension " + std::to_string(c->dim) + " is none of 64, 96, 128, 192, 256";
    if (c->heads < 1 || c->heads > kMostHeads) return "head count out of range";
    if (c->pages < 1) return "the cache has no pages";
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return "null cache array";
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return "the cache's pages are not 16-byte aligned";
    if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(c->fault, 4)) return "an array is not aligned to its values";
    if (b->n < 0 || b->n > kMostSeqs) return "sequence count out of range";
    if (b->rows < 0 || b->rows > kMostRows || b->max_new < 0 || b->max_new > kMostRows) return "rows out of range";
    if (b->max_len < 0 || b->max_len > kMostTokens) return "max_len out of range";
    if (b->table_width < 0 || b->max_len > (int64_t)b->table_width * KK_KV_PAGE) return "max_len exceeds the page table's width";
    if (b->n == 0 || b->rows == 0 || b->max_new == 0) return "";
    if (!b->row_start || !b->len || (!b->table && b->max_len)) return "null batch array";
    if (!aligned(b->row_start, 4) || !aligned(b->len, 4) || !aligned(b->table, 4)) return "an array is not aligned to its values";
    return "";
}

std::string kv_rows_error(const kk_kv_rows* r) {
    if (!r) return "null arguments";
    if (r->type != KK_BF16 && r->type != KK_F16 && r->type != KK_F32) return "unknown type " + std::to_string(r->type);
    if (!r->k || !r->v) return "null array";
    if (!aligned(r->k, value_bytes(r->type)) || !aligned(r->v, value_bytes(r->type))) return "an array is not aligned to its values";
    return "";
}

std::string kv_attention_error(const kk_kv_cache* c, const kk_kv_batch* b, const kk_kv_attention_args* a) {
    const std::string e = kv_batch_error(c, b);
    if (!e.empty()) return e;
    if (!a) return "null arguments";
    if (a->type != KK_BF16 && a->type != KK_F16) return "unknown type " + std::to_string(a->type);
    if (a->heads < 1 || a->heads > kMostHeads || a->heads % c->heads)
        return "query heads (" + std::to_string(a->heads) + ") are no multiple of the cache's (" + std::to_string(c->heads) + ")";
    if (!(a->scale > 0.f && std::isfinite(a->scale))) return "scale must be positive and finite";
    if (a->causal != 0 && a->causal != 1) return "causal is 0 or 1";
    if (a->window < 0 || a->window > kMostTokens) return "window out of range";
    if (a->window && !a->causal) return "a window needs causal";
    if (b->n == 0 || b->rows == 0 || b->max_new == 0) return "";
    if (!a->q || !a->out) return "null array";
    if (a->q == a->out) return "the output is the queries' array";
    if (!aligned(a->q, 2) || !aligned(a->out, 2)) return "an array is not aligned to its values";
    return "";
}

}  // namespace kk

using kk::kGapN;

extern "C" {

int kk_durations_from_logits(const float* logits, int t, float speed, int64_t* out) {
    if (!logits || !out || t < 0 || !(speed > 0.f) || !std::isfinite(speed)) return KK_ERR_INVALID;
    // src/model.rs:90-99 with src/ops.rs:49-51: f32 sigmoid, left-to-right f32 sum, ties to even
    for (int i = 0; i < t; i++) {
        float s = 0.f;
        for (int j = 0; j < 50; j++) {
            volatile float e = std::exp(-logits[i * 50 + j]);
            s = s + 1.0f / (1.0f + (float)e);
        }
        const float d = std::nearbyint(s / speed);
        // `d as i64` in Rust saturates: NaN -> 0, at or past 2^63 -> i64::MAX (the sum is >= 0)
        const int64_t di = std::isnan(d) ? 0 : d >= 9.223372036854775808e18f ? INT64_MAX : (int64_t)d;
        out[i] = di < 1 ? 1 : di;
    }
    return KK_OK;
}

int64_t kk_layout_frames(const int64_t* nfs, int n, int64_t* a_out) {
    if (!nfs || !a_out || n <= 0) return KK_ERR_INVALID;
    int64_t ln = 0;
    for (int b = 0; b < n; b++) {
        if (nfs[b] < 0 || nfs[b] > ((int64_t)1 << 40)) return KK_ERR_INVALID;
        a_out[b] = ln;
        ln += nfs[b] + kGapN;
    }
    return ln;
}

int kk_layout_col_item(int64_t l, const int64_t* start, const int64_t* len, int n, int32_t* col_item) {
    if (!start || !len || !col_item || l < 0) return KK_ERR_INVALID;
    for (int64_t t = 0; t < l; t++) col_item[t] = -1;
    for (int b = 0; b < n; b++) {
        if (start[b] < 0 || len[b] < 0 || start[b] > l || len[b] > l - start[b]) return KK_ERR_INVALID;
        for (int64_t t = start[b]; t < start[b] + len[b]; t++) {
            if (col_item[t] >= 0) return KK_ERR_INVALID;
            col_item[t] = b;
        }
    }
    return KK_OK;
}

int kk_layout_src_row(const int64_t* const* dur, const int32_t* n_tok, int n, const int64_t* tstart, const int64_t* a,
                      int64_t ln, int32_t* src_row) {
    if (!dur || !n_tok || !tstart || !a || !src_row || ln < 0) return KK_ERR_INVALID;
    for (int64_t t = 0; t < ln; t++) src_row[t] = -1;
    for (int b = 0; b < n; b++) {
        if (a[b] < 0 || n_tok[b] < 0 || (n_tok[b] > 0 && !dur[b])) return KK_ERR_INVALID;
        int64_t f = a[b];
        for (int tok = 0; tok < n_tok[b]; tok++)
            for (int64_t r = 0; r < dur[b][tok]; r++) {
                if (f >= ln) return KK_ERR_INVALID;
                src_row[f++] = (int32_t)(tstart[b] + tok);
            }
    }
    return KK_OK;
}

}  // extern "C"
