// Host side of the expert matrices and the operators around them.
#pragma once

#include "model.h"
#include "mx.h"

namespace tinyoai {

// `experts` matrices (or (gate, up) pairs) of one shape in the tiles of mx.h.
struct ExpertMatrix {
  MxMat d{};
  void *mem = nullptr, *infinite = nullptr;
  ExpertMatrix() = default;
  ExpertMatrix(const ExpertMatrix &) = delete;
  ExpertMatrix &operator=(const ExpertMatrix &) = delete;
  ~ExpertMatrix();
  // GGUF-encoded matrices one after another, `nbytes` each of data and (null:
  // no pairs) up; waits for the copies to finish.
  int upload(int32_t dtype, int32_t experts, int64_t rows, int64_t cols, const void *data, const void *up,
             uint64_t nbytes, hipStream_t st);
};

// Refusals: a shape, type or size that no matrices have (`each`: bytes of one
// of them); a product past what the kernels address; another current device than the handle's; misaligned code or
// scale rows.
int check_matrices(int32_t dtype, int32_t experts, int64_t rows, int64_t cols, uint64_t nbytes, int64_t *each);
int check_product(const MxProduct &p);
int check_device(int device, const char *what);
int check_mxfp4_rows(const void *codes, const void *scales);

}  // namespace tinyoai
