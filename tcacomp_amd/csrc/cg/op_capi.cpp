// op_capi.cpp — the C ABI of include/tca_op.h.
#include <exception>
#include <new>
#include <string>

#include "capi_types.h"
#include "operators.h"
#include "tca_op.h"

namespace {

thread_local std::string g_op_error;

}  // namespace

extern "C" {

int tca_op_emit(const char* name, const char* attributes, const char* target, tca_emit_result* out) {
  tca_emit_result_s* r = nullptr;
  try {
    if (out == nullptr || name == nullptr) {
      g_op_error = "op_emit: null argument";
      return TCA_ERR_INVALID;
    }
    *out = nullptr;
    r = new tca_emit_result_s;
    std::string err;
    const auto st = tca::cg::EmitOperator(name, attributes ? attributes : "", target ? target : "gfx950", &r->r, &r->program, &err);
    if (st != tca::cg::OpStatus::Ok) {
      delete r;
      r = nullptr;
      g_op_error = err;
      return st == tca::cg::OpStatus::NoSuchOperator ? TCA_ERR_NOT_FOUND : TCA_ERR_UNSUPPORTED;
    }
    *out = r;
    return TCA_OK;
  } catch (const std::exception& e) {
    delete r;
    try {
      g_op_error = std::string("op_emit: ") + e.what();
    } catch (...) {
      g_op_error.clear();
    }
    return TCA_ERR_INVALID;
  }
}

const char* tca_op_program_name(tca_emit_result r) { return r ? r->program.c_str() : nullptr; }

const char* tca_op_last_error(void) { return g_op_error.c_str(); }

const char* tca_op_list(void) {
  try {
    static const std::string text = tca::cg::ListOperators();
    return text.c_str();
  } catch (...) {
    return "";
  }
}

}  // extern "C"
