// The part of the DLPack in-memory interface (dmlc/dlpack, version 0.x: the unversioned DLManagedTensor every
// array library exchanges) that device arrays need: names, order and codes are the specification's.
#pragma once
#include <stdint.h>

namespace rx {

enum : int32_t { kDLCUDA = 2 };
enum : uint8_t { kDLInt = 0, kDLUInt = 1, kDLFloat = 2, kDLBfloat = 4, kDLBool = 6 };

struct DLDevice {
  int32_t device_type, device_id;
};
struct DLDataType {
  uint8_t code, bits;
  uint16_t lanes;
};
struct DLTensor {
  void* data;
  DLDevice device;
  int32_t ndim;
  DLDataType dtype;
  int64_t *shape, *strides;  // strides in elements; null: row-major
  uint64_t byte_offset;
};
struct DLManagedTensor {
  DLTensor dl_tensor;
  void* manager_ctx;
  void (*deleter)(DLManagedTensor*);
};

}  // namespace rx
