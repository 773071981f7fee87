// Rotary positions of queries and keys in fixed point (the float step of llama-self-attn.py:42-73 in whole numbers; an addition to the class layer).
#pragma once
#include "fr-tensor.hpp"
#include "int-tensor.hpp"

struct RopeConfig {
    double base = 0;              // 10000 in LLaMa-2; 0: no positions
    uint dim = 0;                 // the rotated part of a head, 0: all of it
    bool neighbours = false;      // pairs (2 i, 2 i + 1) instead of (i, i + dim / 2)
    double factor = 1;            // frequencies divided by this ...
    double original = 0;          // ... or, above 0, only those that turn less than `high` times over this many positions (in full below `low`)
    double low = 1, high = 4;
    double magnitude = 1;         // cosines and sines times this
    uint first = 0;               // the first token's position
    uint scale = 1u << 16;        // of the table
};

// The table of a prompt of `tokens` tokens and its use.
class Rotary {
   public:
    Rotary(const RopeConfig& c, uint tokens, uint head_dim);
    // x: [token][head][dim] -> the same, or [head][token][dim]
    FrTensor operator()(const FrTensor& x, uint heads, bool by_head) const;
    void rotate(int32_t* out, const int32_t* x, uint heads, bool by_head, void* flag_dev) const;
    void check() const { flag.check("rotary positions"); }      // whether every element of the field tensors handed in so far, rotated or copied, was a 32-bit integer

   private:
    const RopeConfig c;
    const uint tokens, head_dim, rot;
    IntTensor table;
    ValuesFlag flag;
};
