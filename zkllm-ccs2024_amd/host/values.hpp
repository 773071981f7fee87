// A decoder layer's values without their witness (an addition): what llama_layer returns, computed in int32 by a few kernels, for a caller who needs the layer's
// answer and no proof -- the inputs of all layers before any of them is proved, so that they can be proved on as many devices as there are, or the
// model's answer before its proof.
#pragma once
#include "int-tensor.hpp"
#include "layer.hpp"

class LayerValues {
   public:
    // Lays out what the calls read: the weights' digit planes (shared with the layer's proofs where those keep them), the norms' weights and the activation
    // table in int32.  c and w must outlive it, unmodified (w's planes).
    LayerValues(const LayerConfig& c, const LayerWeights& w);
    ~LayerValues();
    LayerValues(const LayerValues&) = delete;
    LayerValues& operator=(const LayerValues&) = delete;
    // X: tokens x embed_dim in fixed point, any number of tokens.  Element for element llama_layer's output; throws when a value leaves int32 or the
    // activation table, where the proof's own lookups fail as well or its tensors hold larger numbers.
    IntTensor operator()(const IntTensor& X) const;

   private:
    const LayerConfig& c;
    struct Rhs { const void* prepared = nullptr; bool own = false; };
    Rhs q, k, v, o, up, gate, down;
    IntTensor input_norm, post_norm, act;
    Rhs rhs(const FrTensor& weight, uint in_dim, uint out_dim);
    void release();
};
