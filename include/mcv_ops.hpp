/* C++ shim over the mcv_matmul.h C ABI with the reference engine's op names
 * and calling convention (src/csrc/include/minicpmv/ops.h): tensors in,
 * output tensor by reference, a stream last, errors as exceptions.
 *
 * The functions are templates over the caller's tensor type; it needs
 *   void* data() const;  const std::vector<int64_t>& shape() const;
 * which the reference's minicpmv::Tensor provides (tensor.h:56-60), so the
 * engine's call sites keep their arguments.  Unlike the reference, calls do
 * not synchronise the stream unless `sync` is true (ops.cpp:359-377 syncs
 * after every op).  Quantized weights are the library's own packed formats
 * (W4A16Weight / W8A8Weight below), prepared once at load time. */
#ifndef MCV_OPS_HPP
#define MCV_OPS_HPP

#include <cuda_runtime_api.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <vector>

#include "mcv_matmul.h"

namespace mcv_ops {

/* A failed call: the library status and its message (mcv_last_error). */
class Error : public std::runtime_error {
public:
    Error(int status, const std::string& what)
        : std::runtime_error(what + ": " + mcv_status_string(status) + ": " + mcv_last_error()), status_(status) {}
    int status() const { return status_; }

private:
    int status_;
};

inline void check(int status, const char* what) {
    if (status != MCV_OK) throw Error(status, what);
}

inline void finish(cudaStream_t stream, bool sync, const char* what) {
    if (!sync) return;
    const cudaError_t e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

/* mcv-int4 weight of one projection (mcv_w4a16_pack_*_host + one H2D copy
 * per array).  Stands in for W4A16QuantizedWeight (quantized_weight.h:11-17). */
struct W4A16Weight {
    const void* qweight = nullptr;
    const void* scales = nullptr;
    const void* zeros = nullptr;
    int zero_bias = 0;
    int64_t K = 0, N = 0;
};

/* int8 weight [N][K] + fp16 per-channel scales [N] (mcv_w8a8_quantize_weight,
 * w_layout 0).  Stands in for W8A8QuantizedWeight (quantized_weight.h:19-24). */
struct W8A8Weight {
    const void* w_int8 = nullptr;
    const void* w_scale = nullptr;
    int64_t K = 0, N = 0;
};

namespace detail {
template <class T>
void need_rank2(const T& t, const char* what) {
    if (t.shape().size() != 2) throw Error(MCV_ERR_SHAPE, std::string(what) + ": expected a 2-D tensor");
}
}  // namespace detail

/* out [M,N] = x [M,K] . W for the packed int4 weight (the GEMV up to 32 rows,
 * or 64 rows with K <= 4096; the tensor-core GEMM beyond).  ops.h:104-108. */
template <class T>
void matmul_w4a16(const T& x, const W4A16Weight& w, T& out, cudaStream_t stream, bool sync = false) {
    detail::need_rank2(x, "matmul_w4a16");
    const int64_t M = x.shape()[0], K = x.shape()[1];
    if (K != w.K) throw Error(MCV_ERR_SHAPE, "matmul_w4a16: x and weight K differ");
    const int st = (M <= 32 || (M <= 64 && K <= 4096)) ? mcv_w4a16_gemv(x.data(), w.qweight, w.scales, w.zeros, w.zero_bias, out.data(), M, K,
                                           w.N, 128, stream)
                          : mcv_w4a16_gemm(x.data(), w.qweight, w.scales, w.zeros, w.zero_bias, out.data(), M, K,
                                           w.N, 128, stream);
    check(st, "matmul_w4a16");
    finish(stream, sync, "matmul_w4a16");
}

/* The MLP's gate / up projections and their silu_mul in one launch:
 * act [M,N] = silu_mul(x . gate, x . up) (decoder_layer.cpp:1186-1203). */
template <class T>
void matmul_w4a16_gate_up_silu(const T& x, const W4A16Weight& gate, const W4A16Weight& up, T& act,
                               cudaStream_t stream, bool sync = false) {
    detail::need_rank2(x, "matmul_w4a16_gate_up_silu");
    const mcv_w4a16_problem g{nullptr, gate.qweight, gate.scales, gate.zeros, nullptr, static_cast<int32_t>(gate.K),
                              static_cast<int32_t>(gate.N), 128, gate.zero_bias};
    const mcv_w4a16_problem u{nullptr, up.qweight, up.scales, up.zeros, nullptr, static_cast<int32_t>(up.K),
                              static_cast<int32_t>(up.N), 128, up.zero_bias};
    check(mcv_w4a16_gemv_gate_up_silu(x.data(), &g, &u, act.data(), x.shape()[0], stream), "matmul_w4a16_gate_up_silu");
    finish(stream, sync, "matmul_w4a16_gate_up_silu");
}

/* out [M,N] = a [M,K] . B with b stored [N,K] or [K,N], told apart by a's K
 * as the reference does (ops.cpp:165-171): the GEMV for M <= 8, the
 * tensor-core GEMM beyond ([N,K] weights only).  ops.h:19. */
template <class T>
void matmul_b_transposed(const T& a, const T& b, T& out, cudaStream_t stream, bool sync = false) {
    detail::need_rank2(a, "matmul_b_transposed");
    detail::need_rank2(b, "matmul_b_transposed");
    const int64_t M = a.shape()[0], K = a.shape()[1];
    int layout;
    int64_t N;
    if (b.shape()[1] == K) {
        layout = 0, N = b.shape()[0];
    } else if (b.shape()[0] == K) {
        layout = 1, N = b.shape()[1];
    } else {
        throw Error(MCV_ERR_SHAPE, "matmul_b_transposed: K dim mismatch");
    }
    if (M > 8) {
        // the tensor-core GEMM takes [N,K]; a [K,N] weight needs mcv_transpose_f16 once at load time
        if (layout != 0) throw Error(MCV_ERR_SHAPE, "matmul_b_transposed: M > 8 needs the weight as [N,K]");
        check(mcv_gemm_f16(a.data(), b.data(), out.data(), M, K, N, stream), "matmul_b_transposed");
    } else {
        check(mcv_gemv_f16(a.data(), b.data(), out.data(), M, K, N, layout, stream), "matmul_b_transposed");
    }
    finish(stream, sync, "matmul_b_transposed");
}

/* int64 [M] = first-max index of fp16 [M,V] along the last dim.  ops.h:21. */
template <class T>
void argmax_last_dim(const T& self, T& out, cudaStream_t stream, bool sync = false) {
    detail::need_rank2(self, "argmax_last_dim");
    check(mcv_argmax_last_dim_f16(self.data(), out.data(), self.shape()[0], self.shape()[1], stream),
          "argmax_last_dim");
    finish(stream, sync, "argmax_last_dim");
}

/* int32 [M,N] = int8 x [M,K] . int8 w [K,N] (the reference's layout).  ops.h:112-115. */
template <class T>
void matmul_w8a8_i32(const T& x, const T& w, T& out, cudaStream_t stream, bool sync = false) {
    detail::need_rank2(x, "matmul_w8a8_i32");
    detail::need_rank2(w, "matmul_w8a8_i32");
    check(mcv_w8a8_gemm_i32(x.data(), w.data(), out.data(), x.shape()[0], x.shape()[1], w.shape()[1], 1, stream),
          "matmul_w8a8_i32");
    finish(stream, sync, "matmul_w8a8_i32");
}

/* Per-row absmax quantization to int8 + fp16 scales.  ops.h:117-120. */
template <class T>
void w8a8_quantize(const T& x, T& x_int8, T& x_scale, cudaStream_t stream, bool sync = false) {
    detail::need_rank2(x, "w8a8_quantize");
    check(mcv_w8a8_quantize(x.data(), x_int8.data(), x_scale.data(), x.shape()[0], x.shape()[1], stream),
          "w8a8_quantize");
    finish(stream, sync, "w8a8_quantize");
}

/* fp16 out = RN((acc * w_scale) * x_scale).  ops.h:122-126. */
template <class T>
void w8a8_dequant(const T& acc, const T& x_scale, const T& w_scale, T& out, cudaStream_t stream, bool sync = false) {
    detail::need_rank2(acc, "w8a8_dequant");
    check(mcv_w8a8_dequant(acc.data(), x_scale.data(), w_scale.data(), out.data(), acc.shape()[0], acc.shape()[1],
                           stream),
          "w8a8_dequant");
    finish(stream, sync, "w8a8_dequant");
}

/* matmul_decode_w8a8_prequant (decoder_layer.cpp:216-224): int8 x with its
 * fp16 scales (from w8a8_quantize) against a W8A8Weight, int32 GEMV + dequant
 * in one kernel. */
template <class T>
void matmul_decode_w8a8_prequant(const T& x_int8, const T& x_scale, const W8A8Weight& w, T& out, cudaStream_t stream,
                                 bool sync = false) {
    detail::need_rank2(x_int8, "matmul_decode_w8a8_prequant");
    if (x_int8.shape()[1] != w.K) throw Error(MCV_ERR_SHAPE, "matmul_decode_w8a8_prequant: x and weight K differ");
    check(mcv_w8a8_gemv_prequant(x_int8.data(), x_scale.data(), w.w_int8, w.w_scale, out.data(), nullptr,
                                 x_int8.shape()[0], w.K, w.N, stream),
          "matmul_decode_w8a8_prequant");
    finish(stream, sync, "matmul_decode_w8a8_prequant");
}

/* The projection's format chosen like matmul_decode_dispatch
 * (decoder_layer.cpp:226-244); absent formats are nullptr. */
template <class T>
void matmul_decode_dispatch(const T& x, const T* dense_weight, const W4A16Weight* quant_weight,
                            const W8A8Weight* w8_weight, T& out, cudaStream_t stream, bool sync = false) {
    detail::need_rank2(x, "matmul_decode_dispatch");
    detail::need_rank2(out, "matmul_decode_dispatch");
    const int64_t M = x.shape()[0], K = x.shape()[1], N = out.shape()[1];
    mcv_decode_weights f{};
    if (dense_weight) {
        detail::need_rank2(*dense_weight, "matmul_decode_dispatch");
        f.dense = dense_weight->data();
        f.dense_layout = dense_weight->shape()[1] == K ? 0 : 1;
    }
    if (quant_weight) {
        f.w4_qweight = quant_weight->qweight;
        f.w4_scales = quant_weight->scales;
        f.w4_zeros = quant_weight->zeros;
        f.w4_zero_bias = quant_weight->zero_bias;
    }
    if (w8_weight) {
        f.w8_weight = w8_weight->w_int8;
        f.w8_scale = w8_weight->w_scale;
    }
    check(mcv_matmul_decode_dispatch(x.data(), &f, out.data(), M, K, N, stream), "matmul_decode_dispatch");
    finish(stream, sync, "matmul_decode_dispatch");
}

/* Greedy lm_head over fp16 embedding rows [V,K] for one row of x: the fused
 * GEMV + first-max argmax, index read back to the host (one 8-byte copy,
 * then a stream sync) - the device part of lm_head_greedy
 * (language_model.cpp:412-482).  `workspace` holds
 * mcv_lm_head_workspace_size(1) zero-filled bytes; index_dev one int64. */
template <class T>
int64_t lm_head_greedy_index(const T& x, const T& embed, void* workspace, size_t workspace_bytes, void* index_dev,
                             cudaStream_t stream) {
    detail::need_rank2(x, "lm_head_greedy_index");
    detail::need_rank2(embed, "lm_head_greedy_index");
    check(mcv_lm_head_argmax(x.data(), embed.data(), nullptr, index_dev, 1, x.shape()[1], embed.shape()[0], 0, 0,
                             workspace, workspace_bytes, stream),
          "lm_head_greedy_index");
    int64_t idx = -1;
    cudaError_t e = cudaMemcpyAsync(&idx, index_dev, sizeof(idx), cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) throw std::runtime_error(std::string("lm_head_greedy_index: ") + cudaGetErrorString(e));
    return idx;
}

/* lm_head_greedy (language_model.cpp:412-482) as the engine calls it: the raw
 * last hidden state [1,K], the final norm weight [K] (rms_norm of :423 fused
 * into the kernel), the fp16 embedding rows [V,K]; returns the token id. */
template <class T>
int64_t lm_head_greedy(const T& last_hidden, const T& final_norm_w, const T& embed, double rms_epsilon,
                       void* workspace, size_t workspace_bytes, void* index_dev, cudaStream_t stream) {
    detail::need_rank2(last_hidden, "lm_head_greedy");
    detail::need_rank2(embed, "lm_head_greedy");
    if (final_norm_w.shape().size() != 1 || final_norm_w.shape()[0] != last_hidden.shape()[1])
        throw Error(MCV_ERR_SHAPE, "lm_head_greedy: norm weight must be [hidden]");
    check(mcv_lm_head_argmax_rmsnorm(nullptr, last_hidden.data(), final_norm_w.data(), static_cast<float>(rms_epsilon),
                                     0, embed.data(), nullptr, index_dev, 1, last_hidden.shape()[1],
                                     embed.shape()[0], 0, 0, workspace, workspace_bytes, stream),
          "lm_head_greedy");
    int64_t idx = -1;
    cudaError_t e = cudaMemcpyAsync(&idx, index_dev, sizeof(idx), cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) throw std::runtime_error(std::string("lm_head_greedy: ") + cudaGetErrorString(e));
    return idx;
}

/* rms_norm (ops.h / ops.cpp:564-737): the engine's fp16 chain with (1 + gamma). */
template <class T>
void rms_norm(const T& x, const T& gamma, T& out, double epsilon, cudaStream_t stream, bool sync = false) {
    if (x.shape().empty() || x.shape() != out.shape()) throw Error(MCV_ERR_SHAPE, "rms_norm: x/out shape mismatch");
    const int64_t H = x.shape().back();
    if (gamma.shape().size() != 1 || gamma.shape()[0] != H) throw Error(MCV_ERR_SHAPE, "rms_norm: gamma must be [H]");
    int64_t rows = 1;
    for (size_t i = 0; i + 1 < x.shape().size(); ++i) rows *= x.shape()[i];
    check(mcv_rms_norm(x.data(), gamma.data(), out.data(), rows, H, static_cast<float>(epsilon), 0, stream), "rms_norm");
    finish(stream, sync, "rms_norm");
}

/* silu_mul (ops.h:41, ops.cpp:437-456). */
template <class T>
void silu_mul(const T& gate, const T& up, T& out, cudaStream_t stream, bool sync = false) {
    if (gate.shape() != up.shape() || gate.shape() != out.shape()) throw Error(MCV_ERR_SHAPE, "silu_mul shape mismatch");
    int64_t n = 1;
    for (int64_t d : gate.shape()) n *= d;
    check(mcv_silu_mul(gate.data(), up.data(), out.data(), n, stream), "silu_mul");
    finish(stream, sync, "silu_mul");
}

/* The W8A8 branch of lm_head_greedy (language_model.cpp:430-479): int8
 * embedding rows `embed_int8` [V,K] with fp16 per-row scales `embed_scale`
 * (mcv_w8a8_quantize_weight, w_layout 2), x quantized in the kernel; index
 * read back as above. */
template <class T>
int64_t lm_head_greedy_index_w8a8(const T& x, const T& embed_int8, const T& embed_scale, void* workspace,
                                  size_t workspace_bytes, void* index_dev, cudaStream_t stream) {
    detail::need_rank2(x, "lm_head_greedy_index_w8a8");
    detail::need_rank2(embed_int8, "lm_head_greedy_index_w8a8");
    check(mcv_lm_head_argmax_w8a8(x.data(), embed_int8.data(), embed_scale.data(), nullptr, index_dev, 1,
                                  x.shape()[1], embed_int8.shape()[0], 0, workspace, workspace_bytes, stream),
          "lm_head_greedy_index_w8a8");
    int64_t idx = -1;
    cudaError_t e = cudaMemcpyAsync(&idx, index_dev, sizeof(idx), cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) throw std::runtime_error(std::string("lm_head_greedy_index_w8a8: ") + cudaGetErrorString(e));
    return idx;
}

/* ---- Token mixing -------------------------------------------------------
 * Over dense tensors; rows that lie apart (a slice of a wider projection) go
 * through the C calls, whose mcv_rows carry strides. */
namespace detail {
template <class T>
mcv_rows heads_of(const T& t, const char* what) {   /* [tokens, heads, head_dim] */
    if (t.shape().size() != 3) throw Error(MCV_ERR_SHAPE, std::string(what) + ": expected [tokens, heads, head_dim]");
    return mcv_rows{t.data(), t.shape()[1] * t.shape()[2], t.shape()[2]};
}
template <class T>
void need_shape(const T& t, const std::vector<int64_t>& shape, const char* what) {
    if (t.shape() != shape) throw Error(MCV_ERR_SHAPE, std::string(what) + ": shapes do not fit together");
}
}  // namespace detail

/* A layer's paged cache from its fp16 tensors [pages, kv_heads, page_size, head_dim]. */
template <class T>
mcv_kv_cache paged_kv_cache(T& k, T& v) {
    if (k.shape().size() != 4 || k.shape() != v.shape())
        throw Error(MCV_ERR_SHAPE, "paged_kv_cache: k and v must be [pages, kv_heads, page_size, head_dim]");
    const auto& s = k.shape();
    for (int64_t n : s)
        if (n < 1 || n > 0x7fffffff) throw Error(MCV_ERR_SHAPE, "paged_kv_cache: bad dimensions");
    return mcv_kv_cache{k.data(), v.data(), s[1] * s[2] * s[3], static_cast<int32_t>(s[0]), static_cast<int32_t>(s[2]),
                        static_cast<int32_t>(s[1]), static_cast<int32_t>(s[3])};
}

/* out = x with its rotary positions; positions int32 [axes, tokens]. */
template <class T>
void mrope(const T& x, const T& positions, const mcv_mrope_spec& spec, T& out, cudaStream_t stream, bool sync = false) {
    const mcv_rows rows = detail::heads_of(x, "mrope");
    const auto& s = x.shape();
    detail::need_shape(out, s, "mrope");
    detail::need_shape(positions, {spec.axes, s[0]}, "mrope");
    check(mcv_mrope(&rows, out.data(), &spec, positions.data(), s[0], s[1], s[2], stream), "mrope");
    finish(stream, sync, "mrope");
}

/* q_out = q rotated; k rotated and v written to the cache (mcv_mrope_append_kv);
 * `seq` nullptr: token t belongs to row t of page_table [rows, pages]. */
template <class T>
void mrope_append_kv(const T& q, const T& k, const T& v, const T& positions, const mcv_mrope_spec& spec,
                     const mcv_kv_cache& cache, const T& page_table, const T* seq, const T& index, T& q_out,
                     cudaStream_t stream, bool sync = false) {
    const mcv_rows qr = detail::heads_of(q, "mrope_append_kv"), kr = detail::heads_of(k, "mrope_append_kv"),
                   vr = detail::heads_of(v, "mrope_append_kv");
    const int64_t n = q.shape()[0];
    detail::need_shape(q, {n, q.shape()[1], cache.head_dim}, "mrope_append_kv");
    detail::need_shape(k, {n, cache.kv_heads, cache.head_dim}, "mrope_append_kv");
    detail::need_shape(v, k.shape(), "mrope_append_kv");
    detail::need_shape(q_out, q.shape(), "mrope_append_kv");
    detail::need_shape(positions, {spec.axes, n}, "mrope_append_kv");
    detail::need_shape(index, {n}, "mrope_append_kv");
    if (seq) detail::need_shape(*seq, {n}, "mrope_append_kv");
    detail::need_rank2(page_table, "mrope_append_kv");
    check(mcv_mrope_append_kv(&qr, q_out.data(), &kr, &vr, &spec, positions.data(), &cache, page_table.data(),
                              page_table.shape()[0], page_table.shape()[1], seq ? seq->data() : nullptr, index.data(), n,
                              q.shape()[1], stream),
          "mrope_append_kv");
    finish(stream, sync, "mrope_append_kv");
}

/* One new token per sequence over the cache (mcv_paged_attention_decode); `lse`
 * may be nullptr; `workspace` holds mcv_paged_attention_workspace_size bytes,
 * zero-filled once. */
template <class T>
void paged_attention_decode(const T& q, const mcv_kv_cache& cache, const T& page_table, const T& lengths, float scale,
                            T& out, T* lse, void* workspace, size_t workspace_bytes, cudaStream_t stream,
                            bool sync = false) {
    const mcv_rows qr = detail::heads_of(q, "paged_attention_decode");
    const int64_t b = q.shape()[0], heads = q.shape()[1];
    detail::need_shape(q, {b, heads, cache.head_dim}, "paged_attention_decode");
    detail::need_shape(out, q.shape(), "paged_attention_decode");
    detail::need_shape(lengths, {b}, "paged_attention_decode");
    detail::need_rank2(page_table, "paged_attention_decode");
    detail::need_shape(page_table, {b, page_table.shape()[1]}, "paged_attention_decode");
    if (lse) detail::need_shape(*lse, {b, heads}, "paged_attention_decode");
    check(mcv_paged_attention_decode(&qr, &cache, page_table.data(), page_table.shape()[1], lengths.data(), out.data(),
                                     lse ? lse->data() : nullptr, b, heads, scale, workspace, workspace_bytes, stream),
          "paged_attention_decode");
    finish(stream, sync, "paged_attention_decode");
}

namespace detail {
template <class T>
mcv_gated_delta delta_of(const T& q, const T& k, const T& v, const T& g, const T& beta, const T* state_in, T* state_out,
                         const T* state_index, int64_t batch, float scale, float l2_eps, T& out, const char* what) {
    mcv_gated_delta a{};
    a.q = heads_of(q, what), a.k = heads_of(k, what), a.v = heads_of(v, what);
    const int64_t n = q.shape()[0], dk = q.shape()[2], vh = v.shape()[1], dv = v.shape()[2];
    need_shape(k, q.shape(), what);
    need_shape(v, {n, vh, dv}, what);
    need_shape(g, {n, vh}, what);
    need_shape(beta, {n, vh}, what);
    need_shape(out, v.shape(), what);
    const T* any = state_in ? state_in : state_out;
    a.slots = any && !any->shape().empty() ? any->shape()[0] : batch;
    if (state_in) need_shape(*state_in, {a.slots, vh, dk, dv}, what);
    if (state_out) need_shape(*state_out, {a.slots, vh, dk, dv}, what);
    if (state_index) need_shape(*state_index, {batch}, what);
    if (q.shape()[1] > 0x7fffffff || vh > 0x7fffffff || dk > 0x7fffffff || dv > 0x7fffffff)
        throw Error(MCV_ERR_SHAPE, std::string(what) + ": bad dimensions");
    a.g = g.data(), a.beta = beta.data(), a.out = out.data();
    a.state_in = state_in ? state_in->data() : nullptr;
    a.state_out = state_out ? state_out->data() : nullptr;
    a.state_index = state_index ? state_index->data() : nullptr;
    a.k_heads = static_cast<int32_t>(q.shape()[1]), a.v_heads = static_cast<int32_t>(vh);
    a.key_dim = static_cast<int32_t>(dk), a.value_dim = static_cast<int32_t>(dv);
    a.scale = scale, a.l2_eps = l2_eps;
    return a;
}
}  // namespace detail

/* One token per sequence of the gated delta rule (mcv_gated_delta_step);
 * state_out may be state_in; state_index nullptr: sequence b has slot b. */
template <class T>
void gated_delta_step(const T& q, const T& k, const T& v, const T& g, const T& beta, const T& state_in, T& state_out,
                      const T* state_index, float scale, float l2_eps, T& out, cudaStream_t stream, bool sync = false) {
    if (q.shape().empty()) throw Error(MCV_ERR_SHAPE, "gated_delta_step: expected [tokens, heads, head_dim]");
    const int64_t batch = q.shape()[0];
    const mcv_gated_delta a = detail::delta_of(q, k, v, g, beta, &state_in, &state_out, state_index, batch, scale,
                                               l2_eps, out, "gated_delta_step");
    check(mcv_gated_delta_step(&a, batch, stream), "gated_delta_step");
    finish(stream, sync, "gated_delta_step");
}

/* Packed prompts (mcv_gated_delta_prefill); cu_seqlens int32 [batch + 1];
 * state_in, state_out and state_index may be nullptr; `workspace` holds
 * mcv_gated_delta_workspace_size bytes. */
template <class T>
void gated_delta_prefill(const T& q, const T& k, const T& v, const T& g, const T& beta, const T& cu_seqlens,
                         const T* state_in, T* state_out, const T* state_index, float scale, float l2_eps, T& out,
                         void* workspace, size_t workspace_bytes, cudaStream_t stream, bool sync = false) {
    if (cu_seqlens.shape().size() != 1) throw Error(MCV_ERR_SHAPE, "gated_delta_prefill: cu_seqlens must be [batch + 1]");
    const int64_t batch = cu_seqlens.shape()[0] - 1;
    const mcv_gated_delta a = detail::delta_of(q, k, v, g, beta, state_in, state_out, state_index, batch, scale, l2_eps,
                                               out, "gated_delta_prefill");
    check(mcv_gated_delta_prefill(&a, cu_seqlens.data(), q.shape()[0], batch, workspace, workspace_bytes, stream),
          "gated_delta_prefill");
    finish(stream, sync, "gated_delta_prefill");
}

}  // namespace mcv_ops

#endif
