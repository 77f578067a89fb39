// C entry points of the attention operators (include/tierstream_amd/tsa_attn.h): the argument checks, then the launches.
#include <cmath>

#include "attn_launch.hpp"
#include "op_check.hpp"

namespace tsa {
namespace {

constexpr uint32_t kMaxTokens = 1u << 24, kMaxHeads = 1024;

// Rows of heads: present, at their element's alignment; `apart` (outputs): no value in two places.
void check_heads(const char* what, const char* name, const tsa_heads& h, uint64_t tokens, uint64_t dim, uint64_t size, bool apart) {
  REQUIRE(h.heads >= 1 && h.heads <= kMaxHeads, SS_E_INVALID, std::string(what) + ": " + name + " has 1.." + std::to_string(kMaxHeads) + " heads");
  check_array(what, name, h.p, size);
  REQUIRE(h.token_stride < (uint64_t(1) << 40) && h.head_stride < (uint64_t(1) << 40), SS_E_INVALID, std::string(what) + ": the strides of " + name);
  if (!apart) return;
  const bool by_token = (h.heads == 1 || h.head_stride >= dim) && (tokens == 1 || h.token_stride >= (h.heads - 1) * h.head_stride + dim);
  const bool by_head = (tokens == 1 || h.token_stride >= dim) && (h.heads == 1 || h.head_stride >= (tokens - 1) * h.token_stride + dim);
  REQUIRE(by_token || by_head, SS_E_INVALID, std::string(what) + ": the rows of " + name + " overlap");
}

void check_half(const char* what, uint32_t type) {
  REQUIRE(type == TSA_BF16 || type == TSA_F16, SS_E_INVALID, std::string(what) + ": TSA_BF16 or TSA_F16");
}

void check_cache(const char* what, const tsa_cache* c, bool pages) {
  REQUIRE(c != nullptr, SS_E_INVALID, std::string(what) + ": null cache");
  REQUIRE(c->head_dim % 32 == 0 && c->head_dim >= 32 && c->head_dim <= TSA_ATTEND_MAX_HEAD_DIM, SS_E_INVALID, std::string(what) + ": a cache of head_dim 32, 64, 96 or 128");
  REQUIRE(c->kv_heads >= 1 && c->kv_heads <= kMaxHeads, SS_E_INVALID, std::string(what) + ": a cache of 1.." + std::to_string(kMaxHeads) + " heads");
  REQUIRE(c->n_pages < (1u << 25), SS_E_INVALID, std::string(what) + ": below 2^25 pages");
  if (!pages) return;
  REQUIRE(c->pages != nullptr || c->n_pages == 0, SS_E_INVALID, std::string(what) + ": null pages");
  REQUIRE(reinterpret_cast<uintptr_t>(c->pages) % 16 == 0, SS_E_INVALID, std::string(what) + ": pages must be 16-byte aligned");
}

void check_table(const char* what, const void* table, uint64_t stride, uint32_t requests, uint32_t width) {
  REQUIRE(requests <= TSA_CACHE_MAX_REQUESTS, SS_E_INVALID, std::string(what) + ": at most " + std::to_string(TSA_CACHE_MAX_REQUESTS) + " requests");
  REQUIRE(width >= 1 && width < (1u << 25), SS_E_INVALID, std::string(what) + ": a table of 1..2^25 - 1 pages a request");
  check_array(what, "table", table, 4);
  REQUIRE(requests <= 1 || stride >= width, SS_E_INVALID, std::string(what) + ": the rows of table overlap");
  REQUIRE(stride < (uint64_t(1) << 40), SS_E_INVALID, std::string(what) + ": the stride of table");
}

void check_rows(const char* what, const tsa_cache* c, const tsa_cache_rows_args* a, bool out) {
  check_cache(what, c, true);
  REQUIRE(a != nullptr, SS_E_INVALID, std::string(what) + ": null arguments");
  check_half(what, a->type);
  REQUIRE(a->tokens < kMaxTokens, SS_E_INVALID, std::string(what) + ": below 2^24 tokens");
  REQUIRE(uint64_t(a->tokens) * c->kv_heads * c->head_dim < (uint64_t(1) << 33), SS_E_INVALID, std::string(what) + ": tokens x kv_heads x head_dim below 2^33");
  if (a->tokens == 0) return;
  check_heads(what, "k", a->k, a->tokens, c->head_dim, 2, out);
  check_heads(what, "v", a->v, a->tokens, c->head_dim, 2, out);
  REQUIRE(a->k.heads == c->kv_heads && a->v.heads == c->kv_heads, SS_E_INVALID, std::string(what) + ": k and v have the cache's heads");
  check_array(what, "slots", a->slots, 4);
}

// The shape alone (what a workspace's size takes).
void check_attend_shape(const char* what, const tsa_attend_args* a) {
  REQUIRE(a != nullptr, SS_E_INVALID, std::string(what) + ": null arguments");
  check_half(what, a->type);
  REQUIRE(a->head_dim % 8 == 0 && a->head_dim >= 8 && a->head_dim <= TSA_ATTEND_MAX_HEAD_DIM, SS_E_INVALID, std::string(what) + ": head_dim a multiple of 8, 8..128");
  REQUIRE(a->tokens < kMaxTokens && a->k_tokens < kMaxTokens && a->sequences < kMaxTokens, SS_E_INVALID, std::string(what) + ": below 2^24 tokens and sequences");
  REQUIRE(a->q.heads >= 1 && a->q.heads <= kMaxHeads && a->k.heads >= 1 && a->q.heads % a->k.heads == 0 && a->v.heads == a->k.heads, SS_E_INVALID,
          std::string(what) + ": q's heads a multiple of k's and v's");
  REQUIRE(uint64_t(a->tokens) * a->q.heads < (uint64_t(1) << 30) && uint64_t(a->k_tokens) * a->k.heads < (uint64_t(1) << 30) &&
              uint64_t(a->sequences) * a->q.heads < (1u << 23),
          SS_E_INVALID, std::string(what) + ": tokens x heads below 2^30, sequences x heads below 2^23");
  REQUIRE(a->causal <= 1 && std::isfinite(a->scale), SS_E_INVALID, std::string(what) + ": causal 0 or 1, a finite scale");
}

void check_attend(const char* what, const tsa_attend_args* a, bool out) {
  check_attend_shape(what, a);
  REQUIRE(a->first || a->sequences == 1, SS_E_INVALID, std::string(what) + ": without first there is one sequence");
  REQUIRE(a->first || !a->k_first, SS_E_INVALID, std::string(what) + ": k_first without first");
  REQUIRE(!a->first || a->k_first || a->tokens == a->k_tokens, SS_E_INVALID, std::string(what) + ": without k_first there are as many keys as queries");
  REQUIRE(reinterpret_cast<uintptr_t>(a->first) % 4 == 0 && reinterpret_cast<uintptr_t>(a->k_first) % 4 == 0 &&
              reinterpret_cast<uintptr_t>(a->lse) % 4 == 0,
          SS_E_INVALID, std::string(what) + ": first, k_first and lse not aligned to their types");
  if (a->tokens) {
    check_heads(what, "q", a->q, a->tokens, a->head_dim, 2, false);
    check_heads(what, "out", a->out, a->tokens, a->head_dim, 2, out);
    REQUIRE(a->out.heads == a->q.heads, SS_E_INVALID, std::string(what) + ": out has q's heads");
  }
  if (a->k_tokens) {
    check_heads(what, "k", a->k, a->k_tokens, a->head_dim, 2, false);
    check_heads(what, "v", a->v, a->k_tokens, a->head_dim, 2, false);
  }
}

void check_cached_shape(const char* what, const tsa_cache* c, const tsa_attend_cached_args* a) {
  check_cache(what, c, false);
  REQUIRE(a != nullptr, SS_E_INVALID, std::string(what) + ": null arguments");
  check_half(what, a->type);
  REQUIRE(a->q.heads >= 1 && a->q.heads <= kMaxHeads && a->q.heads % c->kv_heads == 0, SS_E_INVALID, std::string(what) + ": q's heads a multiple of the cache's");
  REQUIRE(a->tokens < kMaxTokens && uint64_t(a->tokens) * a->q.heads < (1u << 26), SS_E_INVALID, std::string(what) + ": below 2^24 tokens, tokens x heads below 2^26");
  REQUIRE(a->requests <= TSA_CACHE_MAX_REQUESTS, SS_E_INVALID, std::string(what) + ": at most " + std::to_string(TSA_CACHE_MAX_REQUESTS) + " requests");
  REQUIRE(a->width >= 1 && a->width < (1u << 25), SS_E_INVALID, std::string(what) + ": a table of 1..2^25 - 1 pages a request");
  const uint64_t tiles = (a->requests < a->tokens ? a->requests : a->tokens) + uint64_t(a->tokens) * (a->q.heads / c->kv_heads) / 16;
  REQUIRE(tiles * a->width < (uint64_t(1) << 31), SS_E_INVALID, std::string(what) + ": the tables of all tiles of 16 query rows below 2^31 pages");
}

}  // namespace
}  // namespace tsa

using namespace tsa;

extern "C" {

ss_status tsa_rotary_init(const tsa_rotary_params* p, tsa_rotary* out) {
  return guard([&] {
    const char* const w = "tsa_rotary_init";
    REQUIRE(p != nullptr && out != nullptr, SS_E_INVALID, std::string(w) + ": null arguments");
    REQUIRE(p->rotated >= 2 && p->rotated % 2 == 0 && p->rotated <= 2 * TSA_ROTARY_MAX_PAIRS, SS_E_INVALID, std::string(w) + ": an even number of rotated values, 2..256");
    REQUIRE(p->interleaved <= 1, SS_E_INVALID, std::string(w) + ": interleaved 0 or 1");
    REQUIRE(std::isfinite(p->base) && p->base > 0 && std::isfinite(p->factor) && p->factor > 0 && std::isfinite(float(p->amplitude)), SS_E_INVALID,
            std::string(w) + ": a positive base and factor, an amplitude that 32 bits hold");
    REQUIRE(std::isfinite(p->trained) && p->trained >= 0 && std::isfinite(p->low) && std::isfinite(p->high), SS_E_INVALID, std::string(w) + ": a trained length of 0 or more, finite limits");
    REQUIRE(p->factor == 1 || p->trained == 0 || p->high > p->low, SS_E_INVALID, std::string(w) + ": high above low");
    tsa_rotary r = {};
    r.pairs = p->rotated / 2;
    r.interleaved = p->interleaved;
    r.amplitude = p->amplitude;
    for (uint32_t i = 0; i < r.pairs; ++i) {
      double turns = std::pow(p->base, -2.0 * i / p->rotated) / (2 * M_PI);
      if (p->factor != 1) {
        const double inside = (p->trained * turns - p->low) / (p->high - p->low);
        const double keep = p->trained == 0 || !(inside > 0) ? 0.0 : inside < 1 ? inside : 1.0;
        turns *= keep + (1 - keep) / p->factor;
      }
      REQUIRE(std::isfinite(turns * INT32_MAX), SS_E_INVALID, std::string(w) + ": a base and factor whose angles are numbers");
      r.turns[i] = turns;
    }
    *out = r;
  });
}

ss_status tsa_rotate(const tsa_rotary* r, const tsa_rotate_args* a, void* stream) {
  return guard([&] {
    const char* const w = "tsa_rotate";
    REQUIRE(r != nullptr && a != nullptr, SS_E_INVALID, std::string(w) + ": null arguments");
    REQUIRE(r->pairs >= 1 && r->pairs <= TSA_ROTARY_MAX_PAIRS && r->interleaved <= 1, SS_E_INVALID, std::string(w) + ": a rotary that tsa_rotary_init did not make");
    REQUIRE(a->type == TSA_F32 || a->type == TSA_BF16 || a->type == TSA_F16, SS_E_INVALID, std::string(w) + ": TSA_F32, TSA_BF16 or TSA_F16");
    REQUIRE(a->head_dim >= 2 * r->pairs && a->head_dim <= 1024, SS_E_INVALID, std::string(w) + ": head_dim at least what is rotated, at most 1024");
    REQUIRE(a->backward <= 1 && a->tokens < kMaxTokens, SS_E_INVALID, std::string(w) + ": backward 0 or 1, below 2^24 tokens");
    if (a->tokens == 0) return;
    for (int i = 0; i < 2; ++i) {
      if (i == 1 && a->x[1].heads == 0 && a->y[1].heads == 0) break;
      check_heads(w, i ? "x[1]" : "x[0]", a->x[i], a->tokens, a->head_dim, element(a->type), false);
      check_heads(w, i ? "y[1]" : "y[0]", a->y[i], a->tokens, a->head_dim, element(a->type), true);
      REQUIRE(a->x[i].heads == a->y[i].heads, SS_E_INVALID, std::string(w) + ": y has x's heads");
      REQUIRE(a->x[i].p != a->y[i].p || ((a->tokens == 1 || a->x[i].token_stride == a->y[i].token_stride) &&
                                         (a->x[i].heads == 1 || a->x[i].head_stride == a->y[i].head_stride)),
              SS_E_INVALID, std::string(w) + ": y in x's place has x's strides");
    }
    check_array(w, "positions", a->positions, 4);
    launched(launch_rotate(*r, *a, static_cast<hipStream_t>(stream)), w);
  });
}

ss_status tsa_cache_plan(const tsa_cache_plan_args* a, void* stream) {
  return guard([&] {
    const char* const w = "tsa_cache_plan";
    REQUIRE(a != nullptr, SS_E_INVALID, std::string(w) + ": null arguments");
    REQUIRE(a->rows < kMaxTokens && a->pages < (1u << 25), SS_E_INVALID, std::string(w) + ": below 2^24 rows and 2^25 pages");
    if (a->requests) {
      check_table(w, a->table, a->table_stride, a->requests, a->width);
      check_array(w, "lengths", a->lengths, 4);
      check_array(w, "fresh", a->fresh, 4);
      check_array(w, "ends", a->ends, 4);
    }
    if (a->pages) check_array(w, "free", a->free, 4);
    check_array(w, "n_free", a->n_free, 4);
    check_array(w, "left", a->left, 4);
    check_array(w, "first", a->first, 4);
    check_array(w, "status", a->status, 4);
    if (a->rows) {
      check_array(w, "positions", a->positions, 4);
      check_array(w, "slots", a->slots, 4);
    }
    launched(launch_cache_plan(*a, static_cast<hipStream_t>(stream)), w);
  });
}

ss_status tsa_cache_slots(const tsa_cache_plan_args* a, void* stream) {
  return guard([&] {
    const char* const w = "tsa_cache_slots";
    REQUIRE(a != nullptr, SS_E_INVALID, std::string(w) + ": null arguments");
    REQUIRE(a->rows < kMaxTokens, SS_E_INVALID, std::string(w) + ": below 2^24 rows");
    if (a->rows == 0) return;
    if (a->requests) {
      check_table(w, a->table, a->table_stride, a->requests, a->width);
      check_array(w, "ends", a->ends, 4);
      check_array(w, "first", a->first, 4);
    }
    check_array(w, "positions", a->positions, 4);
    check_array(w, "slots", a->slots, 4);
    launched(launch_cache_slots(*a, static_cast<hipStream_t>(stream)), w);
  });
}

ss_status tsa_cache_store(const tsa_cache* c, const tsa_cache_rows_args* a, void* stream) {
  return guard([&] {
    check_rows("tsa_cache_store", c, a, false);
    if (a->tokens == 0) return;
    launched(launch_cache_store(*c, *a, static_cast<hipStream_t>(stream)), "tsa_cache_store");
  });
}

ss_status tsa_cache_load(const tsa_cache* c, const tsa_cache_rows_args* a, void* stream) {
  return guard([&] {
    check_rows("tsa_cache_load", c, a, true);
    if (a->tokens == 0) return;
    launched(launch_cache_load(*c, *a, static_cast<hipStream_t>(stream)), "tsa_cache_load");
  });
}

uint64_t tsa_attend_cached_workspace(const tsa_cache* c, const tsa_attend_cached_args* a) {
  uint64_t n = 0;
  (void)guard([&] {
    check_cached_shape("tsa_attend_cached_workspace", c, a);
    n = attend_cached_workspace(*c, *a);
  });
  return n;
}

ss_status tsa_attend_cached(const tsa_cache* c, const tsa_attend_cached_args* a, void* workspace, uint64_t workspace_bytes, void* stream) {
  return guard([&] {
    const char* const w = "tsa_attend_cached";
    check_cached_shape(w, c, a);
    check_cache(w, c, true);
    REQUIRE(std::isfinite(a->scale), SS_E_INVALID, std::string(w) + ": a finite scale");
    if (a->tokens == 0 || a->requests == 0) return;
    check_heads(w, "q", a->q, a->tokens, c->head_dim, 2, false);
    check_heads(w, "out", a->out, a->tokens, c->head_dim, 2, true);
    REQUIRE(a->out.heads == a->q.heads, SS_E_INVALID, std::string(w) + ": out has q's heads");
    check_table(w, a->table, a->table_stride, a->requests, a->width);
    check_array(w, "ends", a->ends, 4);
    check_array(w, "first", a->first, 4);
    check_workspace(w, workspace, workspace_bytes, attend_cached_workspace(*c, *a));
    launched(launch_attend_cached(*c, *a, workspace, static_cast<hipStream_t>(stream)), w);
  });
}

ss_status tsa_attend(const tsa_attend_args* a, void* stream) {
  return guard([&] {
    const char* const w = "tsa_attend";
    check_attend(w, a, true);
    if (a->tokens == 0 || a->sequences == 0) return;
    launched(launch_attend(*a, static_cast<hipStream_t>(stream)), w);
  });
}

uint64_t tsa_attend_backward_workspace(const tsa_attend_args* f) {
  uint64_t n = 0;
  (void)guard([&] {
    check_attend_shape("tsa_attend_backward_workspace", f);
    n = attend_backward_workspace(*f);
  });
  return n;
}

ss_status tsa_attend_backward(const tsa_attend_grad_args* a, void* workspace, uint64_t workspace_bytes, void* stream) {
  return guard([&] {
    const char* const w = "tsa_attend_backward";
    REQUIRE(a != nullptr, SS_E_INVALID, std::string(w) + ": null arguments");
    const tsa_attend_args& f = a->f;
    check_attend(w, &f, false);
    REQUIRE((a->dk.p != nullptr) == (a->dv.p != nullptr), SS_E_INVALID, std::string(w) + ": dk and dv are asked for together");
    if (f.tokens) {
      REQUIRE(f.lse != nullptr, SS_E_INVALID, std::string(w) + ": null lse");
      check_heads(w, "dout", a->dout, f.tokens, f.head_dim, 2, false);
      REQUIRE(a->dout.heads == f.q.heads, SS_E_INVALID, std::string(w) + ": dout has q's heads");
      if (a->dq.p) {
        check_heads(w, "dq", a->dq, f.tokens, f.head_dim, 2, true);
        REQUIRE(a->dq.heads == f.q.heads, SS_E_INVALID, std::string(w) + ": dq has q's heads");
      }
    }
    if (f.k_tokens && a->dk.p) {
      check_heads(w, "dk", a->dk, f.k_tokens, f.head_dim, 2, true);
      check_heads(w, "dv", a->dv, f.k_tokens, f.head_dim, 2, true);
      REQUIRE(a->dk.heads == f.k.heads && a->dv.heads == f.k.heads, SS_E_INVALID, std::string(w) + ": dk and dv have k's heads");
    }
    const bool queries = f.tokens && a->dq.p, keys = f.k_tokens && a->dk.p;
    if (f.sequences == 0 || (!queries && !keys)) return;
    check_workspace(w, workspace, workspace_bytes, attend_backward_workspace(f));
    launched(launch_attend_backward(*a, workspace, static_cast<hipStream_t>(stream)), w);
  });
}

}  // extern "C"
