// C entry points of the model operators (include/tierstream_amd/tsa_ops.h): the argument checks, then the launches.
#include <cmath>

#include "op_check.hpp"

namespace tsa {
namespace {

void check_route(const char* what, const tsa_route_args* a) {
  REQUIRE(a != nullptr, SS_E_INVALID, std::string(what) + ": null arguments");
  REQUIRE(a->type == TSA_F32 || a->type == TSA_BF16 || a->type == TSA_F16, SS_E_INVALID, std::string(what) + ": logits of TSA_F32, TSA_BF16 or TSA_F16");
  REQUIRE(a->n_experts >= 1 && a->n_experts <= TSA_ROUTE_MAX_EXPERTS, SS_E_INVALID, std::string(what) + ": 1.." + std::to_string(TSA_ROUTE_MAX_EXPERTS) + " experts");
  REQUIRE(a->top_k >= 1 && a->top_k <= a->n_experts && a->top_k <= TSA_ROUTE_MAX_TOP_K, SS_E_INVALID, std::string(what) + ": top_k 1.." + std::to_string(TSA_ROUTE_MAX_TOP_K) + ", at most the experts");
  REQUIRE(a->renorm <= 1 && std::isfinite(a->scale), SS_E_INVALID, std::string(what) + ": renorm 0 or 1, a finite scale");
}

void check_act(const char* what, uint32_t act, bool none) {
  REQUIRE(act <= TSA_ACT_RELU && (none || act != TSA_ACT_NONE), SS_E_INVALID, std::string(what) + ": unknown activation");
}

void check_linear(const char* what, const tsa_linear_args* a) {
  REQUIRE(a != nullptr, SS_E_INVALID, std::string(what) + ": null arguments");
  REQUIRE(a->x_type == TSA_BF16 || a->x_type == TSA_F16, SS_E_INVALID, std::string(what) + ": x of TSA_BF16 or TSA_F16");
  REQUIRE(a->w_type == a->x_type || a->w_type == TSA_Q4, SS_E_INVALID, std::string(what) + ": weights of x's type or TSA_Q4");
  REQUIRE(a->y_type == a->x_type || a->y_type == TSA_F32, SS_E_INVALID, std::string(what) + ": y of x's type or TSA_F32");
  REQUIRE(a->w_type != TSA_Q4 || a->n_in % kQ4Block == 0, SS_E_INVALID, std::string(what) + ": 4-bit rows hold a multiple of 32 values");
  REQUIRE(a->n_in >= 1, SS_E_INVALID, std::string(what) + ": n_in 0");
  REQUIRE(a->rows < (1u << 24) && a->n_in < (1u << 24) && a->n_out < (1u << 24) && uint64_t(a->rows) * a->n_out < (uint64_t(1) << 37),
          SS_E_INVALID, std::string(what) + ": sizes below 2^24, rows x n_out below 2^37");
  check_act(what, a->act, true);
}

// The experts as the kernels take them. `weights` false: only the shape is looked at.
ExpertMap experts_of(const char* what, const tsa_experts* e, bool weights) {
  REQUIRE(e != nullptr, SS_E_INVALID, std::string(what) + ": null experts");
  REQUIRE(e->n_experts >= 1 && e->n_experts <= TSA_FFN_MAX_EXPERTS, SS_E_INVALID, std::string(what) + ": 1.." + std::to_string(TSA_FFN_MAX_EXPERTS) + " experts");
  REQUIRE(e->d_model >= 1 && e->d_ff >= 1 && e->d_model < (1u << 24) && e->d_ff < (1u << 24), SS_E_INVALID, std::string(what) + ": d_model and d_ff 1..2^24 - 1");
  REQUIRE(e->w_type == TSA_BF16 || e->w_type == TSA_F16 || e->w_type == TSA_Q4, SS_E_INVALID, std::string(what) + ": weights of TSA_BF16, TSA_F16 or TSA_Q4");
  REQUIRE(e->w_type != TSA_Q4 || (e->d_model % kQ4Block == 0 && e->d_ff % kQ4Block == 0), SS_E_INVALID, std::string(what) + ": 4-bit rows hold a multiple of 32 values");
  ExpertMap m;
  m.n = e->n_experts;
  if (!weights) return m;
  const uint64_t align = e->w_type == TSA_Q4 ? 4 : 2;
  const uint64_t bytes[3] = {e->d_ff * weight_row_bytes(e->d_model, e->w_type), e->d_ff * weight_row_bytes(e->d_model, e->w_type),
                             e->d_model * weight_row_bytes(e->d_ff, e->w_type)};
  const int forms = (e->part[0] != nullptr) + (e->table != nullptr) + (e->view != nullptr);
  REQUIRE(forms == 1, SS_E_INVALID, std::string(what) + ": exactly one of part, table and view says where the weights are");
  if (e->part[0]) {
    for (int p = 0; p < 3; ++p) {
      check_array(what, "weights", e->part[p], align);
      REQUIRE(e->part_stride[p] % align == 0 && (e->n_experts == 1 || e->part_stride[p] >= bytes[p]), SS_E_INVALID, std::string(what) + ": the experts' weights overlap");
      m.part[p] = static_cast<const char*>(e->part[p]);
      m.stride[p] = e->part_stride[p];
    }
  } else if (e->table) {
    check_array(what, "table", e->table, 8);
    m.form = 1;
    m.table = e->table;
    for (int p = 1; p < 3; ++p) m.stride[p] = m.stride[p - 1] + bytes[p - 1];
  } else {
    const ss_dg_device_view& v = *e->view;
    REQUIRE(v.struct_size >= offsetof(ss_dg_device_view, absent_err), SS_E_INVALID, std::string(what) + ": a view of another version");
    m.form = 2;
    std::memcpy(&m.view, &v, v.struct_size < sizeof m.view ? v.struct_size : sizeof m.view);
    m.gated = e->gated;
    REQUIRE(v.n_parts == 3 && v.slot_of && v.unit_base && v.abort && e->gated < v.n_gated, SS_E_INVALID,
            std::string(what) + ": a view of three parts and the gated layer");
    for (int p = 0; p < 3; ++p) {
      check_array(what, "weights", v.parts[p].base, align);
      REQUIRE(v.parts[p].bytes == bytes[p] && v.parts[p].stride >= bytes[p] && v.parts[p].stride % align == 0, SS_E_INVALID,
              std::string(what) + ": the view's parts are not gate, up and down of this shape");
    }
  }
  return m;
}

void check_pairs(const char* what, uint32_t rows, uint32_t top_k, const int32_t* ids, const float* weights) {
  REQUIRE(top_k >= 1 && top_k <= TSA_ROUTE_MAX_TOP_K, SS_E_INVALID, std::string(what) + ": top_k 1.." + std::to_string(TSA_ROUTE_MAX_TOP_K));
  REQUIRE(uint64_t(rows) * top_k < (1u << 24), SS_E_INVALID, std::string(what) + ": rows x top_k below 2^24");
  REQUIRE(rows == 0 || ids || top_k == 1, SS_E_INVALID, std::string(what) + ": without ids top_k is 1");
  REQUIRE(reinterpret_cast<uintptr_t>(ids) % 4 == 0 && reinterpret_cast<uintptr_t>(weights) % 4 == 0, SS_E_INVALID,
          std::string(what) + ": ids and weights not aligned to their types");
}

void check_types(const char* what, const tsa_experts* e, uint32_t type, bool q4) {
  REQUIRE(type == TSA_BF16 || type == TSA_F16, SS_E_INVALID, std::string(what) + ": TSA_BF16 or TSA_F16");
  REQUIRE(q4 || e->w_type != TSA_Q4, SS_E_UNSUPPORTED, std::string(what) + ": 4-bit weights have no backward pass");
  REQUIRE(e->w_type == type || e->w_type == TSA_Q4, SS_E_INVALID, std::string(what) + ": weights of x's type or TSA_Q4");
}

}  // namespace
}  // namespace tsa

using namespace tsa;

extern "C" {

ss_status tsa_route(const tsa_route_args* a, void* stream) {
  return guard([&] {
    const char* const w = "tsa_route";
    check_route(w, a);
    if (a->rows == 0) return;
    check_matrix(w, "logits", a->logits, a->rows, a->n_experts, a->logits_stride, element(a->type));
    check_array(w, "ids", a->ids, 4);
    check_array(w, "weights", a->weights, 4);
    launched(launch_route(*a, static_cast<hipStream_t>(stream)), "tsa_route");
  });
}

ss_status tsa_route_backward(const tsa_route_args* a, const float* dweights, void* dlogits, uint64_t dlogits_stride,
                             void* stream) {
  return guard([&] {
    const char* const w = "tsa_route_backward";
    check_route(w, a);
    if (a->rows == 0) return;
    check_matrix(w, "logits", a->logits, a->rows, a->n_experts, a->logits_stride, element(a->type));
    check_matrix(w, "dlogits", dlogits, a->rows, a->n_experts, dlogits_stride, element(a->type));
    check_array(w, "ids", a->ids, 4);
    check_array(w, "dweights", dweights, 4);
    launched(launch_route_backward(*a, dweights, dlogits, dlogits_stride, static_cast<hipStream_t>(stream)),
             "tsa_route_backward");
  });
}

uint64_t tsa_linear_workspace(const tsa_linear_args* a) {
  uint64_t n = 0;
  (void)guard([&] {
    check_linear("tsa_linear_workspace", a);
    n = linear_workspace(*a);
  });
  return n;
}

ss_status tsa_linear(const tsa_linear_args* a, void* workspace, uint64_t workspace_bytes, void* stream) {
  return guard([&] {
    const char* const w = "tsa_linear";
    check_linear(w, a);
    if (a->rows == 0 || a->n_out == 0) return;
    check_matrix(w, "x", a->x, a->rows, a->n_in, a->x_stride, 2);
    if (a->w_type == TSA_Q4) {
      check_array(w, "w", a->w, 4);
      REQUIRE(a->w_stride == a->n_in, SS_E_INVALID, std::string(w) + ": rows of 4-bit weights lie back to back (w_stride = n_in)");
    } else {
      check_matrix(w, "w", a->w, a->n_out, a->n_in, a->w_stride, 2);
    }
    check_matrix(w, "y", a->y, a->rows, a->n_out, a->y_stride, element(a->y_type));
    if (a->residual) check_matrix(w, "residual", a->residual, a->rows, a->n_out, a->residual_stride, element(a->y_type));
    if (a->bias) check_array(w, "bias", a->bias, 2);
    check_workspace(w, workspace, workspace_bytes, linear_workspace(*a));
    launched(launch_linear(*a, workspace, static_cast<hipStream_t>(stream)), "tsa_linear");
  });
}

uint64_t tsa_ffn_workspace(const tsa_experts* e, uint32_t rows, uint32_t top_k) {
  uint64_t n = 0;
  (void)guard([&] {
    experts_of("tsa_ffn_workspace", e, false);
    check_pairs("tsa_ffn_workspace", rows, top_k, reinterpret_cast<const int32_t*>(16), nullptr);
    n = ffn_workspace(e->n_experts, e->d_model, e->d_ff, e->w_type, rows, top_k);
  });
  return n;
}

ss_status tsa_ffn(const tsa_experts* e, const tsa_ffn_args* a, void* workspace, uint64_t workspace_bytes, void* stream) {
  return guard([&] {
    const char* const w = "tsa_ffn";
    REQUIRE(a != nullptr, SS_E_INVALID, std::string(w) + ": null arguments");
    const ExpertMap m = experts_of(w, e, true);
    check_types(w, e, a->type, true);
    check_act(w, a->act, false);
    check_pairs(w, a->rows, a->top_k, a->ids, a->weights);
    if (a->rows == 0) return;
    check_matrix(w, "x", a->x, a->rows, e->d_model, a->x_stride, 2);
    check_matrix(w, "y", a->y, a->rows, e->d_model, a->y_stride, 2);
    if (a->residual) check_matrix(w, "residual", a->residual, a->rows, e->d_model, a->residual_stride, 2);
    check_workspace(w, workspace, workspace_bytes, ffn_workspace(e->n_experts, e->d_model, e->d_ff, e->w_type, a->rows, a->top_k));
    launched(launch_ffn(m, e->d_model, e->d_ff, e->w_type, *a, workspace, static_cast<hipStream_t>(stream)), "tsa_ffn");
  });
}

uint64_t tsa_ffn_backward_workspace(const tsa_experts* e, uint32_t rows, uint32_t top_k) {
  uint64_t n = 0;
  (void)guard([&] {
    experts_of("tsa_ffn_backward_workspace", e, false);
    check_pairs("tsa_ffn_backward_workspace", rows, top_k, reinterpret_cast<const int32_t*>(16), nullptr);
    n = ffn_backward_workspace(e->n_experts, e->d_model, e->d_ff, e->w_type, rows, top_k);
  });
  return n;
}

ss_status tsa_ffn_backward(const tsa_experts* e, const tsa_ffn_grad_args* a, void* workspace, uint64_t workspace_bytes,
                           void* stream) {
  return guard([&] {
    const char* const w = "tsa_ffn_backward";
    REQUIRE(a != nullptr, SS_E_INVALID, std::string(w) + ": null arguments");
    const ExpertMap m = experts_of(w, e, true);
    check_types(w, e, a->type, false);
    check_act(w, a->act, false);
    check_pairs(w, a->rows, a->top_k, a->ids, a->weights);
    REQUIRE((a->dgate != nullptr) == (a->dup != nullptr) && (a->dgate != nullptr) == (a->ddown != nullptr), SS_E_INVALID,
            std::string(w) + ": dgate, dup and ddown are asked for together");
    if (a->rows) {
      check_matrix(w, "x", a->x, a->rows, e->d_model, a->x_stride, 2);
      check_matrix(w, "dy", a->dy, a->rows, e->d_model, a->dy_stride, 2);
      if (a->dx) check_matrix(w, "dx", a->dx, a->rows, e->d_model, a->dx_stride, 2);
      if (a->dweights) check_array(w, "dweights", a->dweights, 4);
    }
    if (a->dgate) {
      check_array(w, "dgate", a->dgate, 2);
      check_array(w, "dup", a->dup, 2);
      check_array(w, "ddown", a->ddown, 2);
    }
    if (a->rows == 0 && !a->dgate) return;
    check_workspace(w, workspace, workspace_bytes, ffn_backward_workspace(e->n_experts, e->d_model, e->d_ff, e->w_type, a->rows, a->top_k));
    launched(launch_ffn_backward(m, e->d_model, e->d_ff, *a, workspace, static_cast<hipStream_t>(stream)), "tsa_ffn_backward");
  });
}

}  // extern "C"
