// Compiled and run by tests/test_cpp_shim_mixing.py: the token-mixing calls of
// the C++ shim (include/mcv_ops.hpp).  Without arguments every call is one that
// the host refuses, so it needs no GPU; with "gpu" a tiny layer step runs and
// its numbers are checked.
#include <cuda_fp16.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "mcv_ops.hpp"

struct Tensor {  // data() / shape() as the engine's
    void* p = nullptr;
    std::vector<int64_t> s;
    void* data() const { return p; }
    const std::vector<int64_t>& shape() const { return s; }
};

template <class F>
int refused(F f, int want, const char* what) {
    try {
        f();
    } catch (const mcv_ops::Error& e) {
        if (e.status() == want) return 0;
        std::printf("%s: status %d, want %d (%s)\n", what, e.status(), want, e.what());
        return 1;
    }
    std::printf("%s: no exception\n", what);
    return 1;
}

int host() {
    using namespace mcv_ops;
    cudaStream_t st = nullptr;
    int bad = 0;
    mcv_mrope_spec spec;
    const int32_t sections[3] = {12, 10, 10};
    check(mcv_mrope_init(&spec, 64, 3, sections, 1, 1e7), "mrope_init");
    Tensor k4{nullptr, {3, 2, 16, 128}}, v4{nullptr, {3, 2, 16, 128}}, v_other{nullptr, {3, 2, 8, 128}};
    bad += refused([&] { paged_kv_cache(k4, v_other); }, MCV_ERR_SHAPE, "caches that differ");
    const mcv_kv_cache cache = paged_kv_cache(k4, v4);
    if (cache.page_stride != 2 * 16 * 128 || cache.page_size != 16 || cache.kv_heads != 2) bad += 1;
    Tensor q{nullptr, {2, 4, 128}}, k{nullptr, {2, 2, 128}}, pos{nullptr, {3, 2}}, pos1{nullptr, {1, 2}}, table{nullptr, {2, 3}},
        idx{nullptr, {2}}, flat{nullptr, {2, 512}}, lse{nullptr, {2, 4}};
    bad += refused([&] { mrope(flat, pos, spec, flat, st); }, MCV_ERR_SHAPE, "2-D rows");
    bad += refused([&] { mrope(q, pos1, spec, q, st); }, MCV_ERR_SHAPE, "positions of one axis");
    bad += refused([&] { mrope(q, pos, spec, q, st); }, MCV_ERR_NULL, "null rows");
    bad += refused([&] { mrope_append_kv<Tensor>(q, q, k, pos, spec, cache, table, nullptr, idx, q, st); }, MCV_ERR_SHAPE,
                   "k with q's heads");
    bad += refused([&] { mrope_append_kv<Tensor>(q, k, k, pos, spec, cache, table, nullptr, idx, q, st); }, MCV_ERR_NULL,
                   "null append");
    bad += refused([&] { paged_attention_decode<Tensor>(q, cache, idx, idx, 1.f, q, &lse, nullptr, 0, st); },
                   MCV_ERR_SHAPE, "1-D page table");
    bad += refused([&] { paged_attention_decode<Tensor>(q, cache, table, idx, 1.f, q, nullptr, nullptr, 0, st); },
                   MCV_ERR_NULL, "null attention");
    Tensor v{nullptr, {2, 4, 64}}, g{nullptr, {2, 4}}, state{nullptr, {5, 4, 128, 64}}, turned{nullptr, {5, 4, 64, 128}},
        cu{nullptr, {2}};
    bad += refused([&] { gated_delta_step<Tensor>(k, k, v, g, g, turned, turned, &idx, 1.f, -1.f, v, st); },
                   MCV_ERR_SHAPE, "state turned round");
    bad += refused([&] { gated_delta_step<Tensor>(k, k, v, g, g, state, state, &idx, 1.f, -1.f, v, st); }, MCV_ERR_NULL,
                   "null step");
    bad += refused([&] { gated_delta_prefill<Tensor>(k, k, v, g, g, table, nullptr, nullptr, nullptr, 1.f, -1.f, v,
                                                     nullptr, 0, st); },
                   MCV_ERR_SHAPE, "2-D bounds");
    bad += refused([&] { gated_delta_prefill<Tensor>(k, k, v, g, g, cu, nullptr, nullptr, nullptr, 1.f, -1.f, v, nullptr,
                                                     0, st); },
                   MCV_ERR_NULL, "null prefill");
    return bad;
}

template <class E>
Tensor device(std::vector<int64_t> shape, const std::vector<E>& values) {
    Tensor t{nullptr, shape};
    int64_t n = 1;
    for (int64_t d : shape) n *= d;
    if (cudaMalloc(&t.p, n * sizeof(E)) != cudaSuccess) throw std::runtime_error("cudaMalloc");
    if (values.empty()) {
        cudaMemset(t.p, 0, n * sizeof(E));
    } else {
        cudaMemcpy(t.p, values.data(), n * sizeof(E), cudaMemcpyHostToDevice);
    }
    return t;
}
template <class E>
std::vector<E> back(const Tensor& t) {
    int64_t n = 1;
    for (int64_t d : t.s) n *= d;
    std::vector<E> v(n);
    if (cudaMemcpy(v.data(), t.p, n * sizeof(E), cudaMemcpyDeviceToHost) != cudaSuccess) throw std::runtime_error("cudaMemcpy");
    return v;
}

// One token at position 1 of one axis with one frequency pair block: q and k are
// ones, so that the rotated pairs are cos - sin and cos + sin; attention over
// the one cached key returns v; the delta rule from a zero state with k = e_0,
// q = 2 e_0 and beta = 1/2 returns v.
int gpu() {
    using namespace mcv_ops;
    cudaStream_t st;
    if (cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking) != cudaSuccess) return 1;
    int bad = 0;
    mcv_mrope_spec spec;
    const int32_t sections[1] = {8};
    check(mcv_mrope_init(&spec, 16, 1, sections, 0, 10000.0), "mrope_init");
    const int D = 64;
    std::vector<__half> ones(D, __float2half(1.f)), vals(D);
    for (int i = 0; i < D; ++i) vals[i] = __float2half(i / 16.f);
    Tensor q = device<__half>({1, 1, D}, ones), v = device<__half>({1, 1, D}, vals), out = device<__half>({1, 1, D}, {});
    Tensor pos = device<int32_t>({1, 1}, {1}), table = device<int32_t>({1, 1}, {1}), index = device<int32_t>({1}, {0}),
           length = device<int32_t>({1}, {1});
    Tensor ck = device<__half>({2, 1, 16, D}, {}), cv = device<__half>({2, 1, 16, D}, {}), rotated = device<__half>({1, 1, D}, {});
    const mcv_kv_cache cache = paged_kv_cache(ck, cv);
    mrope_append_kv<Tensor>(q, q, v, pos, spec, cache, table, nullptr, index, rotated, st, true);
    const auto turned = back<__half>(rotated);
    const auto cached = back<__half>(ck);
    for (int i = 0; i < D; ++i) {
        double want = 1.0;
        if (i < 16) {
            const double a = std::pow(10000.0, -2.0 * (i % 8) / 16);
            want = i < 8 ? std::cos(a) - std::sin(a) : std::cos(a) + std::sin(a);
        }
        // one rounding to fp16 of numbers below 2, and the fp32 rotation before it
        if (std::fabs(__half2float(turned[i]) - want) > 2.0 / 4096 + 1e-6) bad += 1;
        if (std::memcmp(&cached[16 * D + i], &turned[i], 2)) bad += 1;
    }
    size_t bytes = mcv_paged_attention_workspace_size(1, 1, D);
    Tensor ws = device<uint8_t>({static_cast<int64_t>(bytes)}, {}), lse = device<float>({1, 1}, {});
    paged_attention_decode<Tensor>(rotated, cache, table, length, 0.125f, out, &lse, ws.p, bytes, st, true);
    const auto o = back<__half>(out);
    for (int i = 0; i < D; ++i) bad += __half2float(o[i]) != __half2float(vals[i]);
    std::vector<__half> e0(D, __float2half(0.f)), twice = e0;
    e0[0] = __float2half(1.f), twice[0] = __float2half(2.f);
    Tensor dq = device<__half>({1, 1, D}, twice), dk = device<__half>({1, 1, D}, e0);
    Tensor g = device<float>({1, 1}, {-0.25f}), beta = device<float>({1, 1}, {0.5f}), state = device<float>({1, 1, D, D}, {});
    gated_delta_step<Tensor>(dq, dk, v, g, beta, state, state, nullptr, 1.f, -1.f, out, st, true);
    const auto step = back<__half>(out);
    bytes = mcv_gated_delta_workspace_size(1, 1, 1, D, D);
    Tensor ws2 = device<uint8_t>({static_cast<int64_t>(bytes)}, {}), cu = device<int32_t>({2}, {0, 1});
    gated_delta_prefill<Tensor>(dq, dk, v, g, beta, cu, nullptr, &state, nullptr, 1.f, -1.f, out, ws2.p, bytes, st, true);
    const auto prompt = back<__half>(out);
    const auto left = back<float>(state);
    for (int i = 0; i < D; ++i) {
        bad += __half2float(step[i]) != __half2float(vals[i]);
        bad += std::fabs(__half2float(prompt[i]) - __half2float(vals[i])) > std::fabs(__half2float(vals[i])) / 2048;
        bad += std::fabs(left[i] - 0.5f * __half2float(vals[i])) > 1e-6f * std::fabs(__half2float(vals[i]));
    }
    if (mcv_device_errors() != 0) bad += 1;
    return bad;
}

int main(int argc, char**) {
    try {
        const int bad = argc > 1 ? gpu() : host();
        if (bad == 0) std::printf("mixing ok\n");
        return bad != 0;
    } catch (const std::exception& e) {
        std::printf("exception: %s\n", e.what());
        return 1;
    }
}
