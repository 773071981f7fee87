#include "values.hpp"

#include <algorithm>

#include "../../include/zkllm_hip.h"
#include "rotary.hpp"

#define ZKC(call) zk_check((call), #call)

// a weight's planes: those that its products keep (FrTensor::keep_as_matmul_rhs), made now if none has run yet, or a handle of this object's own
LayerValues::Rhs LayerValues::rhs(const FrTensor& weight, uint in_dim, uint out_dim) {
    if (weight.size != in_dim * out_dim) throw std::runtime_error("LayerValues: a weight's size does not match the configuration");
    MatmulRhsCache* rc = weight.rhs_cache.get();
    if (rc) {
        if (rc->prepared && (rc->N != in_dim || rc->P != out_dim)) rc->reset();
        if (!rc->prepared) {
            ZKC(zk_fr_matmul_rhs_prepare(&rc->prepared, weight.gpu_data, in_dim, out_dim, nullptr));
            rc->N = in_dim; rc->P = out_dim;
        }
        return Rhs{rc->prepared, false};
    }
    void* p = nullptr;
    IntTensor ints(weight);
    ZKC(zk_i32_rhs_prepare(&p, ints.gpu_data, in_dim, out_dim, nullptr));
    return Rhs{p, true};
}
LayerValues::LayerValues(const LayerConfig& c, const LayerWeights& w) : c(c), input_norm(w.input_norm.weight), post_norm(w.post_norm.weight), act(w.swiglu_table) {
    if (c.sf_linear > 0x7FFFFFFFu) throw std::runtime_error("LayerValues: sf_linear must lie below 2^31");
    if (c.num_heads == 0 || c.embed_dim % c.num_heads) throw std::runtime_error("LayerValues: embed_dim must be a multiple of num_heads");
    if (input_norm.size != c.embed_dim || post_norm.size != c.embed_dim || act.size != c.swiglu_len) throw std::runtime_error("LayerValues: a weight's size does not match the configuration");
    try {
        const uint E = c.embed_dim, Hd = c.hidden_dim;
        q = rhs(w.q.weight, E, E); k = rhs(w.k.weight, E, E); v = rhs(w.v.weight, E, E); o = rhs(w.o.weight, E, E);
        up = rhs(w.up.weight, E, Hd); gate = rhs(w.gate.weight, E, Hd); down = rhs(w.down.weight, Hd, E);
        const uint d = E / c.num_heads, K = (uint)c.softmax_bs.size();
        if (d <= 256 && K <= 8 && c.softmax_L + c.softmax_M < K && c.softmax_thetas.size() == K - c.softmax_L - c.softmax_M) {
            const int rc = zk_i32_softmax_prepare(&softmax, c.softmax_bs.data(), (int)K, (int)c.softmax_L, (int)c.softmax_M, (double)c.softmax_sf_in, c.softmax_thetas.data(), d, nullptr);
            if (rc != 10001) zk_check(rc, "zk_i32_softmax_prepare");       // 10001: one that it does not take
        }
    } catch (...) { release(); throw; }
}
void LayerValues::release() {
    (void)zk_i32_softmax_free(softmax);
    softmax = nullptr;
    for (Rhs* r : {&q, &k, &v, &o, &up, &gate, &down}) if (r->own) (void)zk_fr_matmul_rhs_free((void*)r->prepared);
}
LayerValues::~LayerValues() { release(); }

void LayerValues::proof_attention(IntTensor& out, const IntTensor& n1, uint T, const ValuesFlag& flag, void* ws, size_t room) const {
    const uint E = c.embed_dim, H = c.num_heads, d = E / H;
    IntTensor proj(T * E);
    // queries, keys and values as stacks [head][token][dim], with their positions; rot = 0 moves the values' heads alone
    FrTensor Qs(T * E), Ks(T * E), Vs(T * E);
    {
        IntTensor stack(T * E);
        std::optional<Rotary> rotary;
        if (c.rope.base != 0) rotary.emplace(c.rope, T, d);
        auto part = [&](FrTensor& stacked, const Rhs& weight, bool positions) {
            ZKC(zk_i32_linear(proj.gpu_data, n1.gpu_data, E, weight.prepared, T, c.sf_linear, ws, room, flag.dev(), nullptr));
            if (positions && rotary) rotary->rotate(stack.gpu_data, proj.gpu_data, H, true, flag.dev());
            else ZKC(zk_i32_rope(stack.gpu_data, d, (size_t)T * d, proj.gpu_data, E, d, T, H, d, 0, 0, nullptr, 0, nullptr, 0, 1, flag.dev(), nullptr));
            ZKC(zk_fr_from_i32(stacked.gpu_data, stack.gpu_data, (size_t)T * E, nullptr));
        };
        part(Qs, q, true);
        part(Ks, k, true);
        part(Vs, v, false);
    }
    // The proof's own attention, without its proof.  As many heads at a time as keep a tensor of scores within 2^28 field elements (8 GiB).
    {
        uint g = H;
        while (g > 1 && ((unsigned long long)g * T * T > (1ull << 28) || H % g)) --g;
        zkAttnStacked attn(g, c.softmax_sf_in, 1UL, c.softmax_bs, c.softmax_L, c.softmax_M, c.softmax_thetas, T, T, d, 1);
        attn.lean_forward = attn.values_only = true;
        FrTensor heads(T * E);
        const uint per = g * T * d;
        for (uint at = 0; at < T * E; at += per) {
            FrTensor sm_in(g * T * T), sm_out(g * T * T), shift(g * T), shifted(0);
            vector<FrTensor> in_seg, out_seg, m_seg;
            FrTensor part = g == H ? attn.compute(Qs, Ks, Vs, sm_in, sm_out, shift, shifted, in_seg, out_seg, m_seg)
                                  : attn.compute(Qs.trunc(at, at + per), Ks.trunc(at, at + per), Vs.trunc(at, at + per), sm_in, sm_out, shift, shifted, in_seg, out_seg, m_seg);
            ZKC(zk_memcpy_d2d(heads.gpu_data + at, part.gpu_data, sizeof(Fr_t) * (size_t)per, nullptr));
        }
        ZKC(zk_i32_from_heads(out.gpu_data, heads.gpu_data, H, T, d, c.sf_attn, c.sf_attn, flag.dev(), nullptr));
    }
}

IntTensor LayerValues::operator()(const IntTensor& X, bool* attention_by_proof) const {
    const uint E = c.embed_dim, Hd = c.hidden_dim, H = c.num_heads, d = E / H, T = X.size / E;
    if (T == 0 || X.size != T * E) throw std::runtime_error("LayerValues: X must be tokens x embed_dim");
    if (T > 0xFFFFu || (unsigned long long)T * std::max(E, Hd) > 0xFFFFFFFFull) throw std::runtime_error("LayerValues: more tokens than a tensor holds scores of");
    ValuesFlag flag;
    const size_t room = std::max(zk_i32_linear_workspace(T, E), zk_i32_linear_workspace(T, Hd));
    DevBuf ws(room ? room : 16);
    auto norm = [&](int32_t* h, int32_t* n, const int32_t* x, const int32_t* b, const int32_t* weight) {
        ZKC(zk_i32_residual_norm(h, n, nullptr, x, E, b, E, nullptr, nullptr, 0, (int32_t)c.sf_linear, weight, T, E, c.rms_eps, c.value_scale, c.sf_linear, flag.dev(), nullptr));
    };
    auto linear = [&](int32_t* out, const int32_t* x, uint in_dim, const Rhs& weight) {
        ZKC(zk_i32_linear(out, x, in_dim, weight.prepared, T, c.sf_linear, ws.p, room, flag.dev(), nullptr));
    };
    IntTensor n1(T * E), x2(T * E), proj(T * E);
    norm(nullptr, n1.gpu_data, X.gpu_data, nullptr, input_norm.gpu_data);
    bool by_proof = softmax == nullptr;
    if (!by_proof) {
        // every token over all of them, as the proof has it: the sequence is the prefix of all its tokens
        IntTensor Q(T * E), K(T * E), V(T * E);
        linear(Q.gpu_data, n1.gpu_data, E, q);
        linear(K.gpu_data, n1.gpu_data, E, k);
        linear(V.gpu_data, n1.gpu_data, E, v);
        std::optional<Rotary> rotary;
        if (c.rope.base != 0) {
            rotary.emplace(c.rope, T, d);
            rotary->rotate(Q.gpu_data, Q.gpu_data, H, false, flag.dev());
            rotary->rotate(K.gpu_data, K.gpu_data, H, false, flag.dev());
        }
        const zk_i32_cache cache{K.gpu_data, V.gpu_data, (size_t)T * E, E, d, T, 1, nullptr, 0};
        const size_t bytes = zk_i32_attention_workspace(T, H, H, d, T, 0, 0);
        DevBuf attn_ws(bytes);
        ValuesFlag scores;
        ZKC(zk_i32_attention(proj.gpu_data, E, d, Q.gpu_data, E, d, T, H, H, d, softmax, &cache, T, nullptr, 0, nullptr, nullptr, 0, 0, c.sf_attn, c.sf_attn, nullptr, attn_ws.p, bytes,
                             scores.dev(), nullptr));
        by_proof = scores.bits() != 0;             // a value that the proof's tensors may hold: its forward pass gives it, or says what is wrong
    }
    if (by_proof) proof_attention(proj, n1, T, flag, ws.p, room);
    if (attention_by_proof) *attention_by_proof = by_proof;
    linear(n1.gpu_data, proj.gpu_data, E, o);
    norm(x2.gpu_data, n1.gpu_data, X.gpu_data, n1.gpu_data, post_norm.gpu_data);
    {
        IntTensor hidden(T * Hd);
        ZKC(zk_i32_gated(hidden.gpu_data, n1.gpu_data, E, gate.prepared, up.prepared, T, c.sf_gate, c.sf_linear, act.gpu_data, c.swiglu_low, c.swiglu_len, c.sf_linear, ws.p, room, flag.dev(), nullptr));
        linear(proj.gpu_data, hidden.gpu_data, Hd, down);
    }
    norm(x2.gpu_data, nullptr, x2.gpu_data, proj.gpu_data, nullptr);
    flag.check("LayerValues");
    return x2;
}
