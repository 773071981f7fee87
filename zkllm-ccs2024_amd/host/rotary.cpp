#include "rotary.hpp"

#include "../../include/zkllm_hip.h"

#define ZKC(call) zk_check((call), #call)

static uint rotated_part(const RopeConfig& c, uint head_dim) {
    const uint rot = c.dim ? c.dim : head_dim;
    if (rot > head_dim || rot % 2) throw std::runtime_error("rotary positions: the rotated part must be even and within the head");
    return rot;
}
static uint table_size(const RopeConfig& c, uint tokens, uint rot) {
    const unsigned long long n = ((unsigned long long)c.first + tokens) * rot;
    if (n > 0xFFFFFFFFull) throw std::runtime_error("rotary positions: the table does not fit a tensor");
    return (uint)n;
}
Rotary::Rotary(const RopeConfig& c, uint tokens, uint head_dim) : c(c), tokens(tokens), head_dim(head_dim), rot(rotated_part(c, head_dim)), table(table_size(c, tokens, rot)) {
    ZKC(zk_rope_table(table.gpu_data, c.first + tokens, rot, c.base, c.factor, c.original, c.low, c.high, c.magnitude, c.scale, nullptr));
}
FrTensor Rotary::operator()(const FrTensor& x, uint heads, bool by_head) const {
    if ((unsigned long long)x.size != (unsigned long long)tokens * heads * head_dim) throw std::runtime_error("rotary positions: incompatible dimensions");
    FrTensor out(x.size);
    const size_t by_token = (size_t)heads * head_dim;
    ZKC(zk_fr_rope(out.gpu_data, by_head ? head_dim : by_token, by_head ? (size_t)tokens * head_dim : head_dim, x.gpu_data, by_token, head_dim, tokens, heads, head_dim, rot, c.neighbours,
                   table.gpu_data, c.first + tokens, nullptr, c.first, c.scale, flag.dev(), nullptr));
    return out;
}
void Rotary::rotate(int32_t* out, const int32_t* x, uint heads, bool by_head, void* flag_dev) const {
    const size_t by_token = (size_t)heads * head_dim;
    ZKC(zk_i32_rope(out, by_head ? head_dim : by_token, by_head ? (size_t)tokens * head_dim : head_dim, x, by_token, head_dim, tokens, heads, head_dim, rot, c.neighbours, table.gpu_data,
                    c.first + tokens, nullptr, c.first, c.scale, flag_dev, nullptr));
}
