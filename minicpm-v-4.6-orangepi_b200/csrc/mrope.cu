// Rotary positions with several axes (time, height, width) on the query and
// key heads, with the keys and values written into a paged cache in the same
// launch: what a full-attention layer does between its projections and the
// attention of the step.
//
// Frequency i of R/2 turns the pair (x_i, x_{i + R/2}) by
// pos[axis(i)] * f_i; the dimensions from R on pass unchanged.  The angle of
// a far position (2^18 and beyond) has no correct digits left in fp32, so it is
// kept in turns, pos * (f_i / 2 pi), in fp64 and reduced to its fraction
// exactly before sin and cos are taken in fp32 (CUDA's sincospif).
//
// Bound by bytes (each row read once and written once; about 3 operations per
// rotated element) as long as the addresses cost little: a row of 64, 128 or 256
// lies across 8, 16 or 32 lanes, so that every access is 16 bytes of a full line
// and the two halves of a pair meet by a shuffle.  A warp has one token: it
// requests the token's rows, computes the R/2 angles with one lane each while they
// are on their way, and keeps the eight pairs of each lane's place for all heads.
// With few tokens up to eight warps share one, a part of the heads each.
// Other head sizes go through a kernel that deals out items.
// 8191 tokens of 8 + 2 + 2 heads of 256 (101 MB, 15.4 us at the copy rate): 19.5 us; in blocks of
// eight warps 25.4, with the places looked up and the angles' entries read behind all rows 21.8,
// with all sizes dealt out as items, whose divisions cost more than the rows, 31.6.
// What is left is latency: a warp's rows, place and angles are one chain of about 5 us, and the registers
// that hold the rows on their way leave an SM 18 to 20 warps.
#include "mixing.cuh"

#include <cmath>

namespace mcv {
unsigned take_mrope_device_error();

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 4;   // tokens per block

constexpr int kWarps = 2;       // of a block of whole rows: small ones take each other's places without a wait
constexpr int kQRows = 8, kKvRows = 2;      // steps of q, and of k and v, on their way at once

static __device__ unsigned g_mrope_dev_error;

struct RopeArgs {
    const __half* q;
    const __half* k;   // null: q alone
    const __half* v;
    __half* q_out;
    __half* ck;
    __half* cv;
    const int32_t* positions;  // [axes][tokens]
    const int32_t* table;
    const int32_t* seq;        // null: token t belongs to row t
    const int32_t* index;
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;
    int64_t page_stride, table_cols;
    int tokens, q_heads, kv_heads, dim, page_size, num_pages, table_rows;
    FastDiv page{1};
    int per_block;             // tokens of a block
    int share;                 // log2 of the warps that share a token
    int in_place;              // q is its own output
};

// Rotates eight pairs: a' = a cos - b sin, b' = b cos + a sin, in fp32, one
// rounding each to the output's fp16.
__device__ __forceinline__ void rotate8(uint4& a, uint4& b, const float2* cs) {
    uint32_t* ap = &a.x;
    uint32_t* bp = &b.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(u32_as_h2(ap[i])), y = __half22float2(u32_as_h2(bp[i]));
        const float2 c0 = cs[2 * i], c1 = cs[2 * i + 1];
        ap[i] = h2_as_u32(__floats2half2_rn(x.x * c0.x - y.x * c0.y, x.y * c1.x - y.y * c1.y));
        bp[i] = h2_as_u32(__floats2half2_rn(y.x * c0.x + x.x * c0.y, y.y * c1.x + x.y * c1.y));
    }
}

// Element offset of the token's slot in head 0 of the cache, -1: not written.
__device__ __forceinline__ int64_t place_of(const RopeArgs& a, int i, int row) {
    if (i < 0) return -1;
    const int page = a.page.div(i);
    int p = -1;
    if (row >= 0 && row < a.table_rows && page < a.table_cols) p = a.table[row * a.table_cols + page];
    if (p >= 0 && p < a.num_pages) return p * a.page_stride + static_cast<int64_t>(i - page * a.page_size) * a.dim;
    atomicOr(&g_mrope_dev_error, kDevErrIndex);
    return -1;
}
__device__ __forceinline__ float2 turn_of(const mcv_mrope_spec& spec, const RopeArgs& a, int tok, int i) {
    // lanes read different entries: as constants one after the other, from memory together (200 tokens 4.7 -> 4.1 us)
    uint32_t axis;
    double f;
    asm("ld.u8 %0, [%1];" : "=r"(axis) : "l"(&spec.axis[i]));
    asm("ld.f64 %0, [%1];" : "=d"(f) : "l"(&spec.turns[i]));
    const double turns = static_cast<double>(a.positions[static_cast<int64_t>(axis) * a.tokens + tok]) * f;
    float s, c;
    sincospif(static_cast<float>(2.0 * (turns - rint(turns))), &s, &c);
    return make_float2(c, s);
}

// One step of rows: this lane's vector `x` and its partner's half, mine cos -+ other
// sin in fp32, one rounding to the output's fp16 (s carries the sign).
__device__ __forceinline__ void turn_vector(uint4& x, bool turn, int partner, const float (&c)[8], const float (&s)[8]) {
    uint32_t* xp = &x.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t other = __shfl_sync(0xffffffffu, xp[i], partner);
        const float2 m = __half22float2(u32_as_h2(xp[i])), o = __half22float2(u32_as_h2(other));
        const uint32_t y = h2_as_u32(__floats2half2_rn(m.x * c[2 * i] + o.x * s[2 * i], m.y * c[2 * i + 1] + o.y * s[2 * i + 1]));
        xp[i] = turn ? y : xp[i];
    }
}

// BLOCKS resident: 8 leave a thread the 128 registers that hold all its rows on their way (200 tokens of 16 + 2 + 2
// heads 4.1 us, with 9 4.5); 9 hide more of the tokens' latency when there are many (8191 tokens 19.5 us, with 8 21.6).
template <int VECS, int BLOCKS>
__global__ void __launch_bounds__(kWarps * 32, BLOCKS) mrope_rows_kernel(const __grid_constant__ mcv_mrope_spec spec, const RopeArgs a) {
    constexpr int kPer = 32 / VECS;      // rows of a step
    __shared__ float2 turns[kWarps][VECS * 4];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned id = blockIdx.x * kWarps + warp;     // fewer than 2^29 tokens by at most eight warps
    const int tok = static_cast<int>(id >> a.share), mine = id & ((1 << a.share) - 1);
    if (tok >= a.tokens) return;
    const int sub = lane / VECS, vec = lane % VECS, step = kPer << a.share;
    const int half = spec.rotary_dim / 2, nrot = half / 8;
    const bool turned = vec < 2 * nrot, first = vec < nrot;

    // rows q0 + r step of q, and so of k and v, whose steps the sharing warps take on from q's
    const int q0 = mine * kPer + sub;
    const int q_heads = a.in_place && !turned ? 0 : a.q_heads;      // what passes in place is there already
    const uint4* qp = reinterpret_cast<const uint4*>(a.q + tok * a.q_ts + q0 * a.q_hs) + vec;
    const int64_t qs = step * a.q_hs / 8;
    const int index = a.k ? a.index[tok] : -1, row = a.k && a.seq ? a.seq[tok] : tok;
    // plain loads: in place other warps write rows in the same 32-byte sectors, and a preceding kernel may still write q, k
    // and v while this one starts, both of which the read-only path does not allow
    uint4 xq[kQRows], xk[kKvRows], xv[kKvRows];
#pragma unroll
    for (int r = 0; r < kQRows; ++r) xq[r] = q0 + r * step < q_heads ? qp[r * qs] : make_uint4(0, 0, 0, 0);
    const uint4 *kp = nullptr, *vp = nullptr;
    int64_t ks = 0, vs = 0, place = -1;
    const int shift = (a.q_heads + kPer - 1) / kPer, kv0 = ((mine - shift) & ((1 << a.share) - 1)) * kPer + sub;
    if (a.k) {
        place = place_of(a, index, row);
        kp = reinterpret_cast<const uint4*>(a.k + tok * a.k_ts + kv0 * a.k_hs) + vec;
        vp = reinterpret_cast<const uint4*>(a.v + tok * a.v_ts + kv0 * a.v_hs) + vec;
        ks = step * a.k_hs / 8;
        vs = step * a.v_hs / 8;
#pragma unroll
        for (int r = 0; r < kKvRows; ++r) {
            const bool there = kv0 + r * step < a.kv_heads;
            xk[r] = there ? kp[r * ks] : make_uint4(0, 0, 0, 0);
            xv[r] = there ? vp[r * vs] : make_uint4(0, 0, 0, 0);
        }
    }
    for (int i = lane; i < half; i += 32) turns[warp][i] = turn_of(spec, a, tok, i);
    __syncwarp();
    const int partner = turned ? (first ? lane + nrot : lane - nrot) : lane;
    float c[8] = {}, s[8] = {};
    if (turned) {
        const float4* from = reinterpret_cast<const float4*>(&turns[warp][(first ? vec : vec - nrot) * 8]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 y = from[i];
            c[2 * i] = y.x, c[2 * i + 1] = y.z;
            s[2 * i] = first ? -y.y : y.y, s[2 * i + 1] = first ? -y.w : y.w;
        }
    }
    uint4* op = reinterpret_cast<uint4*>(a.q_out + tok * a.o_ts + q0 * a.o_hs) + vec;
    const int64_t os = step * a.o_hs / 8;
    for (int base = 0;;) {
#pragma unroll
        for (int r = 0; r < kQRows; ++r) {
            turn_vector(xq[r], turned, partner, c, s);
            if (q0 + base + r * step < q_heads) op[r * os] = xq[r];
        }
        base += kQRows * step;
        if (base >= a.q_heads) break;
        qp += kQRows * qs;
        op += kQRows * os;
#pragma unroll
        for (int r = 0; r < kQRows; ++r) xq[r] = q0 + base + r * step < q_heads ? qp[r * qs] : make_uint4(0, 0, 0, 0);
    }
    if (place < 0) return;
    const int64_t head = static_cast<int64_t>(a.page_size) * a.dim, cs = step * head / 8;
    uint4* kc = reinterpret_cast<uint4*>(a.ck + place + kv0 * head) + vec;
    uint4* vc = reinterpret_cast<uint4*>(a.cv + place + kv0 * head) + vec;
    for (int base = 0;;) {
#pragma unroll
        for (int r = 0; r < kKvRows; ++r) {
            turn_vector(xk[r], turned, partner, c, s);
            if (kv0 + base + r * step < a.kv_heads) {
                kc[r * cs] = xk[r];
                vc[r * cs] = xv[r];
            }
        }
        base += kKvRows * step;
        if (base >= a.kv_heads) break;
        kp += kKvRows * ks, vp += kKvRows * vs, kc += kKvRows * cs, vc += kKvRows * cs;
#pragma unroll
        for (int r = 0; r < kKvRows; ++r) {
            const bool there = kv0 + base + r * step < a.kv_heads;
            xk[r] = there ? kp[r * ks] : make_uint4(0, 0, 0, 0);
            xv[r] = there ? vp[r * vs] : make_uint4(0, 0, 0, 0);
        }
    }
}

__global__ void __launch_bounds__(kThreads) mrope_kernel(const __grid_constant__ mcv_mrope_spec spec, RopeArgs a) {
    __shared__ float2 cs[kMaxTokens][MCV_MROPE_MAX_FREQS];
    __shared__ int64_t place[kMaxTokens];   // element offset of the token's slot in head 0, -1: not written
    pdl_trigger();
    pdl_wait();
    const int half = spec.rotary_dim / 2;
    const int t0 = blockIdx.x * a.per_block;
    const int nt = min(a.per_block, a.tokens - t0);
    if (a.k && threadIdx.x >= kThreads - nt) {
        const int t = kThreads - 1 - threadIdx.x;
        place[t] = place_of(a, a.index[t0 + t], a.seq ? a.seq[t0 + t] : t0 + t);
    }
    for (int j = threadIdx.x; j < nt * half; j += kThreads) {
        const int t = j / half, i = j - t * half;
        cs[t][i] = turn_of(spec, a, t0 + t, i);
    }
    __syncthreads();

    const int nrot = half / 8;                                 // rotated items of a head
    const int items = nrot + (a.dim - spec.rotary_dim) / 8;    // and those that pass
    const int heads = a.q_heads + (a.k ? 2 * a.kv_heads : 0);
    const int per_token = heads * items;
    for (int j = threadIdx.x; j < nt * per_token; j += kThreads) {
        const int t = j / per_token;
        const int r = j - t * per_token;
        const int h = r / items, i = r - h * items;
        const int64_t tok = t0 + t;
        const __half* src;
        __half* dst;
        bool turn = true;
        if (h < a.q_heads) {
            src = a.q + tok * a.q_ts + h * a.q_hs;
            dst = a.q_out + tok * a.o_ts + h * a.o_hs;
            if (a.in_place && i >= nrot) continue;
        } else {
            if (place[t] < 0) continue;
            const bool key = h < a.q_heads + a.kv_heads;
            const int kh = h - a.q_heads - (key ? 0 : a.kv_heads);
            src = key ? a.k + tok * a.k_ts + kh * a.k_hs : a.v + tok * a.v_ts + kh * a.v_hs;
            dst = (key ? a.ck : a.cv) + place[t] + static_cast<int64_t>(kh) * a.page_size * a.dim;
            turn = key;
        }
        const uint4* s4 = reinterpret_cast<const uint4*>(src);
        uint4* d4 = reinterpret_cast<uint4*>(dst);
        if (i < nrot) {
            uint4 x = s4[i], y = s4[i + nrot];
            if (turn) rotate8(x, y, &cs[t][i * 8]);
            d4[i] = x;
            d4[i + nrot] = y;
        } else {
            d4[i + nrot] = s4[i + nrot];
        }
    }
}

int check_spec(const char* who, const mcv_mrope_spec* s, int64_t dim) {
    if (!s) return fail(MCV_ERR_NULL, std::string(who) + ": null rope specification");
    if (s->rotary_dim < 16 || s->rotary_dim > 2 * MCV_MROPE_MAX_FREQS || s->rotary_dim % 16 || s->rotary_dim > dim)
        return fail(MCV_ERR_SHAPE, std::string(who) + ": rotary_dim must be a multiple of 16, at most head_dim and 256");
    if (s->axes < 1 || s->axes > 4) return fail(MCV_ERR_VALUE, std::string(who) + ": 1 to 4 axes");
    for (int i = 0; i < s->rotary_dim / 2; ++i)
        if (s->axis[i] >= s->axes) return fail(MCV_ERR_VALUE, std::string(who) + ": frequency with an axis beyond the last");
    return MCV_OK;
}

// Rotating in place needs rows that do not share memory.
int check_in_place(const char* who, const mcv_rows* x, int64_t tokens, int64_t heads, int64_t dim) {
    const bool token_major = x->token_stride >= (heads - 1) * x->head_stride + dim;
    const bool head_major = x->token_stride >= dim && x->head_stride >= (tokens - 1) * x->token_stride + dim;
    if (tokens > 1 && !token_major && !head_major)
        return fail(MCV_ERR_SHAPE, std::string(who) + ": rows rotated in place must not overlap");
    return MCV_OK;
}

int launch_mrope(const mcv_mrope_spec& spec, RopeArgs& a, cudaStream_t stream) {
    const int64_t sms = sm_count();
    if (a.dim == 64 || a.dim == 128 || a.dim == 256) {
        // eight warps a token while they all run at once, else as many as have their rows on their way at once
        const int per = 256 / a.dim, q_steps = (a.q_heads + per - 1) / per, kv_steps = a.k ? (a.kv_heads + per - 1) / per : 0;
        a.share = 0;
        while (a.share < 3 && (q_steps > kQRows << a.share || kv_steps > kKvRows << a.share)) ++a.share;
        if (static_cast<int64_t>(a.tokens) * 8 <= sms * 8 * kWarps) a.share = 3;
        const unsigned grid = static_cast<unsigned>(((static_cast<int64_t>(a.tokens) << a.share) + kWarps - 1) / kWarps);
        if (grid > sms * 8)
            return launch(a.dim == 64 ? mrope_rows_kernel<8, 9> : (a.dim == 128 ? mrope_rows_kernel<16, 9> : mrope_rows_kernel<32, 9>),
                          dim3(grid), dim3(kWarps * 32), 0, stream, spec, a);
        return launch(a.dim == 64 ? mrope_rows_kernel<8, 8> : (a.dim == 128 ? mrope_rows_kernel<16, 8> : mrope_rows_kernel<32, 8>),
                      dim3(grid), dim3(kWarps * 32), 0, stream, spec, a);
    }
    // one token a block while that fills the SMs less than twice, else four, which share the block's set-up
    a.per_block = a.tokens <= 8 * sms ? 1 : kMaxTokens;
    const unsigned grid = static_cast<unsigned>((a.tokens + a.per_block - 1) / a.per_block);
    return launch(mrope_kernel, dim3(grid), dim3(kThreads), 0, stream, spec, a);
}

}  // namespace

int check_rows(const char* who, const char* what, const mcv_rows* r, int64_t heads, int64_t dim) {
    if (!r || !r->data) return fail(MCV_ERR_NULL, std::string(who) + ": null " + what);
    if (!aligned16(r->data)) return fail(MCV_ERR_ALIGN, std::string(who) + ": " + what + " must be 16-byte aligned");
    if (r->token_stride % 8 || r->head_stride % 8)
        return fail(MCV_ERR_ALIGN, std::string(who) + ": strides of " + what + " must be multiples of 8 elements");
    if (r->token_stride < 0 || r->head_stride < 0 || (heads > 1 && r->head_stride < dim))
        return fail(MCV_ERR_SHAPE, std::string(who) + ": strides of " + what + " make rows overlap");
    return MCV_OK;
}

int check_kv_cache(const char* who, const mcv_kv_cache* c) {
    if (!c || !c->k || !c->v) return fail(MCV_ERR_NULL, std::string(who) + ": null cache");
    if (!aligned16(c->k) || !aligned16(c->v)) return fail(MCV_ERR_ALIGN, std::string(who) + ": cache must be 16-byte aligned");
    if (c->num_pages < 1 || c->page_size < 1 || c->kv_heads < 1 || c->kv_heads > 4096 || c->head_dim < 16 ||
        c->head_dim > 1024 || c->head_dim % 8)
        return fail(MCV_ERR_SHAPE, std::string(who) + ": bad cache dimensions");
    if (c->page_stride % 8) return fail(MCV_ERR_ALIGN, std::string(who) + ": page stride must be a multiple of 8 elements");
    if (c->page_stride < static_cast<int64_t>(c->kv_heads) * c->page_size * c->head_dim)
        return fail(MCV_ERR_SHAPE, std::string(who) + ": page stride smaller than a page");
    return MCV_OK;
}

unsigned take_mrope_device_error() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_mrope_dev_error, sizeof(v)) != cudaSuccess) return ~0u;
    if (v) cudaMemcpyToSymbol(g_mrope_dev_error, &zero, sizeof(zero));
    return v;
}

}  // namespace mcv

using namespace mcv;

extern "C" {

int mcv_mrope_init(mcv_mrope_spec* spec, int rotary_dim, int axes, const int32_t* sections, int interleaved,
                   double theta) {
    if (!spec || !sections) return fail(MCV_ERR_NULL, "mrope_init: null pointer");
    if (rotary_dim < 16 || rotary_dim > 2 * MCV_MROPE_MAX_FREQS || rotary_dim % 16)
        return fail(MCV_ERR_SHAPE, "mrope_init: rotary_dim must be a multiple of 16, at most 256");
    if (axes < 1 || axes > 4) return fail(MCV_ERR_VALUE, "mrope_init: 1 to 4 axes");
    if (!(theta > 1.0) || std::isinf(theta)) return fail(MCV_ERR_VALUE, "mrope_init: theta must be above 1");
    const int half = rotary_dim / 2;
    int64_t sum = 0;
    for (int a = 0; a < axes; ++a) {
        if (sections[a] < 0) return fail(MCV_ERR_VALUE, "mrope_init: negative section");
        sum += sections[a];
    }
    if (sum != half) return fail(MCV_ERR_SHAPE, "mrope_init: sections must add up to rotary_dim / 2");
    // interleaved: axis a > 0 owns frequencies a, a + axes, ... and all of them must exist
    if (interleaved)
        for (int a = 1; a < axes; ++a)
            if (sections[a] > 0 && a + static_cast<int64_t>(axes) * (sections[a] - 1) >= half)
                return fail(MCV_ERR_SHAPE, "mrope_init: an interleaved section runs past rotary_dim / 2");
    spec->rotary_dim = rotary_dim;
    spec->axes = axes;
    const double two_pi = 6.283185307179586476925286766559;
    for (int i = 0; i < MCV_MROPE_MAX_FREQS; ++i) {
        spec->turns[i] = i < half ? std::pow(theta, -static_cast<double>(i) / half) / two_pi : 0.0;
        int axis = 0;
        if (i < half) {
            if (interleaved) {
                const int a = i % axes;
                axis = a && i < axes * sections[a] ? a : 0;
            } else {
                for (int at = sections[0]; axis < axes - 1 && i >= at;) at += sections[++axis];
            }
        }
        spec->axis[i] = static_cast<uint8_t>(axis);
    }
    return MCV_OK;
}

int mcv_mrope(const mcv_rows* x, void* out, const mcv_mrope_spec* spec, const void* positions, int64_t tokens,
              int64_t heads, int64_t head_dim, mcv_stream_t stream) {
    int st = check_rows("mrope", "x", x, heads, head_dim);
    if (st) return st;
    if (!out || !positions) return fail(MCV_ERR_NULL, "mrope: null out or positions");
    if (!aligned16(out)) return fail(MCV_ERR_ALIGN, "mrope: out must be 16-byte aligned");
    if (tokens < 1 || tokens > 0x7fffffffLL / 4 || heads < 1 || heads > 4096 || head_dim < 16 || head_dim > 1024 || head_dim % 8)
        return fail(MCV_ERR_SHAPE, "mrope: bad tokens, heads or head_dim");
    if ((st = check_spec("mrope", spec, head_dim))) return st;
    if (x->data == out && (st = check_in_place("mrope", x, tokens, heads, head_dim))) return st;
    RopeArgs a{};
    a.q = static_cast<const __half*>(x->data);
    a.q_out = static_cast<__half*>(out);
    a.q_ts = x->token_stride;
    a.q_hs = x->head_stride;
    a.in_place = x->data == out;
    // in place, out has x's strides; else it is dense
    a.o_hs = a.in_place ? a.q_hs : head_dim;
    a.o_ts = a.in_place ? a.q_ts : heads * head_dim;
    a.positions = static_cast<const int32_t*>(positions);
    a.tokens = static_cast<int>(tokens);
    a.q_heads = static_cast<int>(heads);
    a.dim = static_cast<int>(head_dim);
    return launch_mrope(*spec, a, static_cast<cudaStream_t>(stream));
}

int mcv_mrope_append_kv(const mcv_rows* q, void* q_out, const mcv_rows* k, const mcv_rows* v,
                        const mcv_mrope_spec* spec, const void* positions, const mcv_kv_cache* cache,
                        const void* page_table, int64_t table_rows, int64_t table_cols, const void* seq,
                        const void* index, int64_t tokens, int64_t q_heads, mcv_stream_t stream) {
    int st = check_kv_cache("mrope_append_kv", cache);
    if (st) return st;
    const int64_t dim = cache->head_dim;
    if ((st = check_rows("mrope_append_kv", "q", q, q_heads, dim))) return st;
    if ((st = check_rows("mrope_append_kv", "k", k, cache->kv_heads, dim))) return st;
    if ((st = check_rows("mrope_append_kv", "v", v, cache->kv_heads, dim))) return st;
    if (!q_out || !positions || !page_table || !index) return fail(MCV_ERR_NULL, "mrope_append_kv: null pointer");
    if (!aligned16(q_out)) return fail(MCV_ERR_ALIGN, "mrope_append_kv: q_out must be 16-byte aligned");
    if (tokens < 1 || tokens > 0x7fffffffLL / 4 || q_heads < 1 || q_heads > 4096)
        return fail(MCV_ERR_SHAPE, "mrope_append_kv: bad tokens or q_heads");
    if (table_rows < 1 || table_rows > 0x7fffffffLL || table_cols < 1 || table_cols > 0x7fffffffLL)
        return fail(MCV_ERR_SHAPE, "mrope_append_kv: bad page table dimensions");
    if (!seq && table_rows < tokens)
        return fail(MCV_ERR_SHAPE, "mrope_append_kv: one table row per token is needed without seq");
    if ((st = check_spec("mrope_append_kv", spec, dim))) return st;
    if (q->data == q_out && (st = check_in_place("mrope_append_kv", q, tokens, q_heads, dim))) return st;
    RopeArgs a{};
    a.q = static_cast<const __half*>(q->data);
    a.k = static_cast<const __half*>(k->data);
    a.v = static_cast<const __half*>(v->data);
    a.q_out = static_cast<__half*>(q_out);
    a.ck = static_cast<__half*>(cache->k);
    a.cv = static_cast<__half*>(cache->v);
    a.positions = static_cast<const int32_t*>(positions);
    a.table = static_cast<const int32_t*>(page_table);
    a.seq = static_cast<const int32_t*>(seq);
    a.index = static_cast<const int32_t*>(index);
    a.q_ts = q->token_stride, a.q_hs = q->head_stride;
    a.k_ts = k->token_stride, a.k_hs = k->head_stride;
    a.v_ts = v->token_stride, a.v_hs = v->head_stride;
    a.in_place = q->data == q_out;
    a.o_hs = a.in_place ? a.q_hs : dim;
    a.o_ts = a.in_place ? a.q_ts : q_heads * dim;
    a.page_stride = cache->page_stride;
    a.table_cols = table_cols;
    a.tokens = static_cast<int>(tokens);
    a.q_heads = static_cast<int>(q_heads);
    a.kv_heads = cache->kv_heads;
    a.dim = cache->head_dim;
    a.page_size = cache->page_size;
    a.page = FastDiv(static_cast<uint32_t>(cache->page_size));
    a.num_pages = cache->num_pages;
    a.table_rows = static_cast<int>(table_rows);
    return launch_mrope(*spec, a, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
