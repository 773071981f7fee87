// IntTensor: owning device array of int32 in fixed point, the form the activation and parameter files hold (an addition; the reference keeps
// every tensor as field elements; files are read and written by FrTensor).  What LayerValues computes with; an eighth of a field element's bytes.
#pragma once
#include <cstdint>
#include "fr-tensor.hpp"

class IntTensor {
   public:
    int32_t* gpu_data;
    const uint size;

    explicit IntTensor(uint size);
    explicit IntTensor(const FrTensor& t);         // throws when an element is no 32-bit integer
    IntTensor(IntTensor&& t) noexcept;
    IntTensor(const IntTensor&) = delete;
    IntTensor& operator=(const IntTensor&) = delete;
    ~IntTensor();

    FrTensor to_fr() const;
};

// The flag that the int32 entry points raise (ZK_VALUES_*): cleared when made, read once the work that may raise it is queued.
class ValuesFlag {
   public:
    ValuesFlag();
    void* dev() const { return buf.p; }
    void check(const char* what) const;            // waits; throws when a bit is raised

   private:
    DevBuf buf;
};
