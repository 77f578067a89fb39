// Argument checks that the operators' C entry points share: done on the host, before any launch.
#pragma once

#include <hip/hip_runtime_api.h>

#include <string>

#include "common.hpp"
#include "op_launch.hpp"

namespace tsa {

// require() of a check on the way of every call: the message is made only for a refusal.
#define REQUIRE(ok, status, message)    \
  do {                                  \
    if (!(ok)) fail(status, message);   \
  } while (0)

inline void launched(int e, const char* what) {
  if (e != 0) fail(SS_E_BACKEND, std::string(what) + ": " + hipGetErrorString(hipError_t(e)));
}

inline uint64_t element(uint32_t type) { return type == TSA_F32 ? 4 : 2; }

// A matrix of rows x n: present, at its element's alignment, its rows apart.
inline void check_matrix(const char* what, const char* name, const void* p, uint64_t rows, uint64_t n, uint64_t stride,
                         uint64_t size) {
  REQUIRE(p != nullptr, SS_E_INVALID, std::string(what) + ": null " + name);
  REQUIRE(reinterpret_cast<uintptr_t>(p) % size == 0, SS_E_INVALID, std::string(what) + ": " + name + " not aligned to its type");
  REQUIRE(rows <= 1 || stride >= n, SS_E_INVALID, std::string(what) + ": the rows of " + name + " overlap");
  REQUIRE(stride < (uint64_t(1) << 40), SS_E_INVALID, std::string(what) + ": the stride of " + name);
}

inline void check_array(const char* what, const char* name, const void* p, uint64_t size) {
  REQUIRE(p != nullptr, SS_E_INVALID, std::string(what) + ": null " + name);
  REQUIRE(reinterpret_cast<uintptr_t>(p) % size == 0, SS_E_INVALID, std::string(what) + ": " + name + " not aligned to its type");
}

inline void check_workspace(const char* what, const void* p, uint64_t have, uint64_t need) {
  REQUIRE(have >= need && (need == 0 || p), SS_E_INVALID,
          std::string(what) + ": the workspace holds " + std::to_string(p ? have : 0) + " of " + std::to_string(need) + " bytes");
  REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, SS_E_INVALID, std::string(what) + ": the workspace must be 16-byte aligned");
}

}  // namespace tsa
