#include "int-tensor.hpp"

#include "../../include/zkllm_hip.h"

#define ZKC(call) zk_check((call), #call)

static int32_t* int_alloc(uint size) {
    void* p = nullptr;
    ZKC(zk_malloc(&p, sizeof(int32_t) * (size_t)(size ? size : 1)));
    return (int32_t*)p;
}
IntTensor::IntTensor(uint size) : gpu_data(int_alloc(size)), size(size) {}
IntTensor::IntTensor(const FrTensor& t) : IntTensor(t.size) { ZKC(zk_i32_from_heads(gpu_data, t.gpu_data, 1, 1, t.size, 1, 1, nullptr, nullptr)); }
IntTensor::IntTensor(IntTensor&& t) noexcept : gpu_data(t.gpu_data), size(t.size) { t.gpu_data = nullptr; }
IntTensor::~IntTensor() { if (gpu_data) (void)zk_free(gpu_data); }

FrTensor IntTensor::to_fr() const {
    FrTensor out(size);
    ZKC(zk_fr_from_i32(out.gpu_data, gpu_data, size, nullptr));
    return out;
}

ValuesFlag::ValuesFlag() : buf(4) { ZKC(zk_i32_fill(buf.p, 0, 1, nullptr)); }
void ValuesFlag::check(const char* what) const {
    uint32_t bits = 0;
    ZKC(zk_memcpy_d2h(&bits, buf.p, 4, nullptr));
    if (bits & ZK_VALUES_TABLE) throw std::runtime_error(string(what) + ": an activation lies outside the table of function values");
    if (bits & ZK_VALUES_POSITION) throw std::runtime_error(string(what) + ": a position lies outside the table of angles");
    if (bits) throw std::runtime_error(string(what) + ": a value does not fit");
}
