// What the learner's operators share: element types, vector accesses of any alignment, the host-side error and device plumbing.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mbt_env.h"

// mbt_env.hip: the thread-local message behind mbt_last_error(), and the "is it a gfx950" check
__attribute__((visibility("hidden"))) int mbt_set_error(int code, const char* fmt, ...);
__attribute__((visibility("hidden"))) int mbt_device_check(int device);

namespace mbt_learning {

#define LEARNING_HIP_TRY(expr)                                                                                                  \
  do {                                                                                                                          \
    hipError_t e_ = (expr);                                                                                                     \
    if (e_ != hipSuccess) return mbt_set_error(MBT_ERR_HIP, "%s failed: %s", #expr, hipGetErrorString(e_));                     \
  } while (0)

// Makes `device` current for one call and puts the caller's device back: the operators take tensors of any device, whichever is current.
class DeviceScope {
 public:
  int enter(int device) {
    const int rc = mbt_device_check(device);
    if (rc != MBT_OK) return rc;
    LEARNING_HIP_TRY(hipGetDevice(&before_));
    if (before_ != device) {
      LEARNING_HIP_TRY(hipSetDevice(device));
      changed_ = true;
    }
    return MBT_OK;
  }
  ~DeviceScope() {
    if (changed_) (void)hipSetDevice(before_);
  }

 private:
  int before_ = 0;
  bool changed_ = false;
};

inline int launch_status(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? MBT_OK : mbt_set_error(MBT_ERR_HIP, "%s: launch failed: %s", what, hipGetErrorString(e));
}

typedef __bf16 bfloat16;
typedef _Float16 float16;

// V elements at an address that only has the alignment of ONE element (a row of odd length starts anywhere): one wide access, which global
// memory takes at any alignment.
template <typename E, int V>
struct __attribute__((packed, aligned(alignof(E)))) Pack {
  E e[V];
};

template <typename E, int V>
__device__ __forceinline__ Pack<E, V> load_pack(const E* p) {
  Pack<E, V> v;
  __builtin_memcpy(&v, p, sizeof v);
  return v;
}
template <typename E, int V>
__device__ __forceinline__ void store_pack(E* p, const Pack<E, V>& v) {
  __builtin_memcpy(p, &v, sizeof v);
}

// The same past the caches, for arrays that are larger than they and read or written once: what they would drive out is worth more.  Accesses of a
// size that is no power of two are ordinary ones.
template <int BYTES, int ALIGNED>
struct Words;
template <int ALIGNED>
struct Words<4, ALIGNED> {
  typedef uint32_t type;
};
#define LEARNING_WORDS(BYTES, ALIGNED)                                                          \
  template <>                                                                                   \
  struct Words<BYTES, ALIGNED> {                                                                \
    typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4), aligned(ALIGNED)));        \
  };
LEARNING_WORDS(8, 4)
LEARNING_WORDS(8, 2)
LEARNING_WORDS(16, 4)
LEARNING_WORDS(16, 2)
template <typename E, int V>
__device__ __forceinline__ Pack<E, V> stream_load_pack(const E* p) {
  constexpr int kBytes = sizeof(E) * V;
  Pack<E, V> v;
  if constexpr ((kBytes == 4 && alignof(E) == 4) || kBytes == 8 || kBytes == 16) {
    typedef typename Words<kBytes, alignof(E)>::type words;
    const words w = __builtin_nontemporal_load(reinterpret_cast<const words*>(p));
    __builtin_memcpy(&v, &w, kBytes);
  } else {
    v = load_pack<E, V>(p);
  }
  return v;
}
template <typename E, int V>
__device__ __forceinline__ void stream_store_pack(E* p, const Pack<E, V>& v) {
  constexpr int kBytes = sizeof(E) * V;
  if constexpr ((kBytes == 4 && alignof(E) == 4) || kBytes == 8 || kBytes == 16) {
    typedef typename Words<kBytes, alignof(E)>::type words;
    words w;
    __builtin_memcpy(&w, &v, kBytes);
    __builtin_nontemporal_store(w, reinterpret_cast<words*>(p));
  } else {
    store_pack<E, V>(p, v);
  }
}

inline size_t dtype_size(int dtype) { return dtype == MBT_FLOAT32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype == MBT_FLOAT32 || dtype == MBT_BFLOAT16 || dtype == MBT_FLOAT16; }

}  // namespace mbt_learning
