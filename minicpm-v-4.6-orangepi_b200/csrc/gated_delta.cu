// The gated delta rule of the linear-attention layers.  Per value head, with a
// state S [Dk][Dv] (fp32) and per token q, k (Dk), v (Dv), a log decay g and a
// write strength beta:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q,
// with q and k divided by sqrt(sum x^2 + eps) first when asked.  Value heads
// h * v_heads / k_heads ... share key head h.
#include "mixing.cuh"

#include <cmath>

namespace mcv {
unsigned take_gated_delta_device_error();

namespace {

static __device__ unsigned g_gated_delta_dev_error;

struct DeltaArgs {
    const __half* q;
    const __half* k;
    const __half* v;
    const float* g;
    const float* beta;
    __half* out;
    const float* state_in;    // null: zeros
    float* state_out;         // null: not kept
    const int32_t* index;     // null: sequence b has slot b
    const int32_t* cu;        // null: sequence b is token b
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
    int batch, tokens, slots, v_heads, share, dv;
    float scale, l2_eps;
};

// The tokens and the state slot of sequence b; false: nothing to do.
__device__ __forceinline__ bool sequence(const DeltaArgs& a, int b, int& begin, int& end, int& slot) {
    slot = a.index ? a.index[b] : b;
    begin = a.cu ? a.cu[b] : b;
    end = a.cu ? a.cu[b + 1] : b + 1;
    if (slot < 0) return false;
    if (slot >= a.slots || begin < 0 || end < begin || end > a.tokens) {
        if (threadIdx.x == 0) atomicOr(&g_gated_delta_dev_error, kDevErrIndex);
        return false;
    }
    return true;
}

// ---- one token after the other -------------------------------------------------
//
// Bound by the state's bytes (8 Dk Dv per head and token step, read and written
// once; 7 operations per element).  A warp keeps 16 columns of a head's state in
// registers - 8 lane groups take every eighth row, four lanes a 64-byte row
// piece - and works without any block-wide step: the products S^T k and S^T q
// are taken in one pass over the old state, since
// S_new^T q = e^g S^T q + (k.q) u.
constexpr int kCols = 16;

template <int DK>
__global__ void __launch_bounds__(256) recurrent_kernel(const DeltaArgs a) {
    constexpr int kRows = DK / 8;    // rows of a lane
    constexpr int kPer = DK / 32;    // q, k elements of a lane
    __shared__ float2 kq[8][DK];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = (blockIdx.x * (blockDim.x >> 5) + warp) * kCols + (lane & 3) * 4;
    const int rg = lane >> 2;
    const int b = blockIdx.z, h = blockIdx.y;
    int begin, end, slot;
    if (!sequence(a, b, begin, end, slot) || col >= a.dv) return;
    const int64_t at = ((static_cast<int64_t>(slot) * a.v_heads + h) * DK + rg) * a.dv + col;
    float4 s[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
        s[i] = a.state_in ? *reinterpret_cast<const float4*>(a.state_in + at + static_cast<int64_t>(i) * 8 * a.dv)
                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const int kh = h / a.share;
    for (int64_t t = begin; t < end; ++t) {
        const __half* qp = a.q + t * a.q_ts + kh * a.q_hs + lane * kPer;
        const __half* kp = a.k + t * a.k_ts + kh * a.k_hs + lane * kPer;
        const uint2 vv = *reinterpret_cast<const uint2*>(a.v + t * a.v_ts + h * a.v_hs + col);
        const float decay = expf(a.g[t * a.v_heads + h]), beta = a.beta[t * a.v_heads + h];
        float qx[kPer], kx[kPer];
#pragma unroll
        for (int i = 0; i < kPer; i += 2) {
            const float2 x = __half22float2(*reinterpret_cast<const __half2*>(qp + i));
            const float2 y = __half22float2(*reinterpret_cast<const __half2*>(kp + i));
            qx[i] = x.x, qx[i + 1] = x.y, kx[i] = y.x, kx[i + 1] = y.y;
        }
        float qq = 0.0f, kk = 0.0f, qk = 0.0f;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            qq += qx[i] * qx[i];
            kk += kx[i] * kx[i];
            qk += qx[i] * kx[i];
        }
        qk = warp_sum(qk);
        float rq = a.scale, rk = 1.0f;
        if (a.l2_eps >= 0.0f) {
            rq *= 1.0f / sqrtf(warp_sum(qq) + a.l2_eps);
            rk = 1.0f / sqrtf(warp_sum(kk) + a.l2_eps);
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kPer; ++i) kq[warp][lane * kPer + i] = make_float2(kx[i] * rk, qx[i] * rq);
        __syncwarp();
        float ks[4] = {}, qs[4] = {};
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float2 w = kq[warp][rg + 8 * i];
            ks[0] += w.x * s[i].x, ks[1] += w.x * s[i].y, ks[2] += w.x * s[i].z, ks[3] += w.x * s[i].w;
            qs[0] += w.y * s[i].x, qs[1] += w.y * s[i].y, qs[2] += w.y * s[i].z, qs[3] += w.y * s[i].w;
        }
        const float2 v01 = __half22float2(u32_as_h2(vv.x)), v23 = __half22float2(u32_as_h2(vv.y));
        const float v[4] = {v01.x, v01.y, v23.x, v23.y};
        float u[4], o[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                ks[c] += __shfl_xor_sync(0xffffffffu, ks[c], x);
                qs[c] += __shfl_xor_sync(0xffffffffu, qs[c], x);
            }
            u[c] = beta * (v[c] - decay * ks[c]);
            o[c] = decay * qs[c] + qk * rq * rk * u[c];
        }
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            const float k = kq[warp][rg + 8 * i].x;
            s[i].x = decay * s[i].x + k * u[0];
            s[i].y = decay * s[i].y + k * u[1];
            s[i].z = decay * s[i].z + k * u[2];
            s[i].w = decay * s[i].w + k * u[3];
        }
        if (rg == 0)
            *reinterpret_cast<uint2*>(a.out + (t * a.v_heads + h) * a.dv + col) =
                make_uint2(h2_as_u32(__floats2half2_rn(o[0], o[1])), h2_as_u32(__floats2half2_rn(o[2], o[3])));
    }
    if (a.state_out) {
#pragma unroll
        for (int i = 0; i < kRows; ++i)
            *reinterpret_cast<float4*>(a.state_out + at + static_cast<int64_t>(i) * 8 * a.dv) = s[i];
    }
}

int run_recurrent(const DeltaArgs& a, int dk, cudaStream_t stream) {
    // warps of a block: a head's columns, fewer while the blocks would not fill the SMs
    const int cols = a.dv / kCols;
    int warps = cols < 8 ? cols : 8;
    while (warps > 1 && static_cast<int64_t>(a.batch) * a.v_heads * ((cols + warps - 1) / warps) < 2 * sm_count()) warps /= 2;
    const dim3 grid((cols + warps - 1) / warps, a.v_heads, a.batch);
    return launch(dk == 128 ? recurrent_kernel<128> : recurrent_kernel<64>, grid, dim3(warps * 32), 0, stream, a);
}

int fill_args(const char* who, const mcv_gated_delta* p, int64_t tokens, int64_t batch, DeltaArgs& a) {
    if (!p || !p->g || !p->beta || !p->out) return fail(MCV_ERR_NULL, std::string(who) + ": null pointer");
    if (p->key_dim != 64 && p->key_dim != 128) return fail(MCV_ERR_SHAPE, std::string(who) + ": key_dim must be 64 or 128");
    if (p->value_dim < 16 || p->value_dim > 1024 || p->value_dim % 16)
        return fail(MCV_ERR_SHAPE, std::string(who) + ": value_dim must be a multiple of 16 up to 1024");
    if (p->k_heads < 1 || p->v_heads < 1 || p->v_heads > 65535 || p->v_heads % p->k_heads)
        return fail(MCV_ERR_SHAPE, std::string(who) + ": v_heads must be a multiple of k_heads");
    if (batch < 1 || batch > 65535) return fail(MCV_ERR_SHAPE, std::string(who) + ": batch must be 1..65535");
    if (tokens < 1 || tokens > 0x7fffffffLL - 64) return fail(MCV_ERR_SHAPE, std::string(who) + ": bad number of tokens");
    if (p->slots < 1 || p->slots > 0x7fffffffLL || (!p->state_index && p->slots < batch))
        return fail(MCV_ERR_SHAPE, std::string(who) + ": one state slot per sequence is needed without an index");
    int st = check_rows(who, "q", &p->q, p->k_heads, p->key_dim);
    if (st) return st;
    if ((st = check_rows(who, "k", &p->k, p->k_heads, p->key_dim))) return st;
    if ((st = check_rows(who, "v", &p->v, p->v_heads, p->value_dim))) return st;
    if (!aligned16(p->out) || !aligned16(p->state_in) || !aligned16(p->state_out))
        return fail(MCV_ERR_ALIGN, std::string(who) + ": out and states must be 16-byte aligned");
    if (!(std::fabs(p->scale) <= 3.0e38f) || p->l2_eps != p->l2_eps)
        return fail(MCV_ERR_VALUE, std::string(who) + ": scale and l2_eps must be numbers");
    a.q = static_cast<const __half*>(p->q.data);
    a.k = static_cast<const __half*>(p->k.data);
    a.v = static_cast<const __half*>(p->v.data);
    a.g = static_cast<const float*>(p->g);
    a.beta = static_cast<const float*>(p->beta);
    a.out = static_cast<__half*>(p->out);
    a.state_in = static_cast<const float*>(p->state_in);
    a.state_out = static_cast<float*>(p->state_out);
    a.index = static_cast<const int32_t*>(p->state_index);
    a.cu = nullptr;
    a.q_ts = p->q.token_stride, a.q_hs = p->q.head_stride;
    a.k_ts = p->k.token_stride, a.k_hs = p->k.head_stride;
    a.v_ts = p->v.token_stride, a.v_hs = p->v.head_stride;
    a.batch = static_cast<int>(batch);
    a.tokens = static_cast<int>(tokens);
    a.slots = static_cast<int>(p->slots);
    a.v_heads = p->v_heads;
    a.share = p->v_heads / p->k_heads;
    a.dv = p->value_dim;
    a.scale = p->scale;
    a.l2_eps = p->l2_eps;
    return MCV_OK;
}

}  // namespace

unsigned take_gated_delta_device_error() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_gated_delta_dev_error, sizeof(v)) != cudaSuccess) return ~0u;
    if (v) cudaMemcpyToSymbol(g_gated_delta_dev_error, &zero, sizeof(zero));
    return v;
}

}  // namespace mcv

using namespace mcv;

extern "C" {

int mcv_gated_delta_step(const mcv_gated_delta* args, int64_t batch, mcv_stream_t stream) {
    DeltaArgs a;
    int st = fill_args("gated_delta_step", args, batch, batch, a);
    if (st) return st;
    if (!a.state_in || !a.state_out) return fail(MCV_ERR_NULL, "gated_delta_step: null state");
    return run_recurrent(a, args->key_dim, static_cast<cudaStream_t>(stream));
}

size_t mcv_gated_delta_workspace_size(int64_t tokens, int64_t batch, int64_t v_heads, int64_t key_dim,
                                      int64_t value_dim) {
    if (tokens < 1 || batch < 1 || v_heads < 1 || (key_dim != 64 && key_dim != 128) || value_dim < 16) return 0;
    return 16;
}

int mcv_gated_delta_prefill(const mcv_gated_delta* args, const void* cu_seqlens, int64_t tokens, int64_t batch,
                            void* workspace, size_t workspace_bytes, mcv_stream_t stream) {
    DeltaArgs a;
    int st = fill_args("gated_delta_prefill", args, tokens, batch, a);
    if (st) return st;
    if (!cu_seqlens) return fail(MCV_ERR_NULL, "gated_delta_prefill: null cu_seqlens");
    if (!workspace || workspace_bytes < mcv_gated_delta_workspace_size(tokens, batch, a.v_heads, args->key_dim, a.dv))
        return fail(MCV_ERR_WORKSPACE, "gated_delta_prefill: workspace missing or too small");
    if (!aligned16(workspace)) return fail(MCV_ERR_ALIGN, "gated_delta_prefill: workspace must be 16-byte aligned");
    a.cu = static_cast<const int32_t*>(cu_seqlens);
    return run_recurrent(a, args->key_dim, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
