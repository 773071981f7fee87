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
    // attention_by_proof (may be null) receives whether the proof's forward pass computed the attention: for heads and softmaxes that zk_i32_attention does not take, and
    // where that raised its flag.
    IntTensor operator()(const IntTensor& X, bool* attention_by_proof = nullptr) const;

   private:
    const LayerConfig& c;
    struct Rhs { const void* prepared = nullptr; bool own = false; };
    Rhs q, k, v, o, up, gate, down;
    IntTensor input_norm, post_norm, act;
    void* softmax = nullptr;       // null where the heads or the softmax are none that zk_i32_attention takes: the proof's own forward pass then
    Rhs rhs(const FrTensor& weight, uint in_dim, uint out_dim);
    void proof_attention(IntTensor& out, const IntTensor& normed, uint tokens, const ValuesFlag& flag, void* ws, size_t room) const;
    void release();
};
