// The gated delta rule of the linear-attention layers.  Per value head, with a
// state S [Dk][Dv] (fp32) and per token q, k (Dk), v (Dv), a log decay g and a
// write strength beta:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q,
// with q and k divided by sqrt(sum x^2 + eps) first when asked.  Value heads
// h * v_heads / k_heads ... share key head h.
#include "mixing.cuh"
#include "tcgen05.cuh"

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

// ---- prompts, in chunks of 64 tokens -----------------------------------------------
//
// With G_i the decay summed up to token i of a chunk, S0 the state before it
// and r the norms' reciprocals, the written rows u of the chunk solve
//   (I + A) U = diag(beta) (V - diag(e^G r_k) K S0),
//   A_ij = beta_i e^(G_i - G_j) r_ki r_kj k_i.k_j   (j < i),
// and O = scale diag(e^G r_q) Q S0 + P U with P_ij = scale e^(G_i - G_j) r_qi r_kj q_i.k_j
// (j <= i), S' = e^G_C S0 + K^T diag(e^(G_C - G_j) r_kj) U.
//
// With T = (I + A)^-1 diag(beta): U = T R for R = V - diag(e^G r_k) K S0, and so
// O = scale diag(e^G r_q) Q S0 + (P T) R.  chunk_kernel makes T and P T, which do
// not need the state, for all chunks at once; walk_kernel then takes the chunks
// of a sequence one after the other.
//
// Everything that has a 16-bit exact operand (K, Q as stored; norms, decays and
// scales are applied to results in fp32) runs on the fp16 tensor MMA with fp32
// accumulation.  The other operands (S, T, P T, R, U) are split as hi + 2^-11 lo,
// both fp16, the lo products in accumulators of their own: 22 bits of each
// value, down to an absolute 2^-36, so results keep fp32's accuracy where
// a single fp16 operand would leave 2^-11.  (State values and written rows are
// below fp16's 65504 then; with |k| <= 1, beta <= 1 and g <= 0 they are bounded by
// the state's start and the sum of |v|.)
constexpr int kChunk = 64;
constexpr float kLo = 2048.0f, kLoInv = 1.0f / 2048.0f;

__device__ __forceinline__ void split_scaled(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = h2_as_u32(h);
    lo = h2_as_u32(__floats2half2_rn((x - f.x) * kLo, (y - f.y) * kLo));
}

// One chunk's share of the workspace: T (rows 0-63) over P T (rows 64-127), hi and
// lo, as the shared-memory image of an MMA operand (rows of 128 bytes, 16-byte
// pieces exchanged by the row's low bits: the 128-byte swizzle), and the scales.
struct Chunk {
    __half tp[2][128 * kChunk];
    float ck[kChunk];                // e^G r_k
    float cq[kChunk];                // scale e^G r_q
    float cs[kChunk];                // e^(G_C - G) r_k
    float keep;                      // e^G_C
    float pad[63];
};
static_assert(sizeof(Chunk) == 33 * 1024, "a chunk is copied whole");

// Byte offset of element (r, c) in a tile of 128-byte rows under the 128-byte swizzle.
__device__ __forceinline__ uint32_t sw128(int r, int c) { return r * 128 + ((((c >> 3) ^ r) & 7) << 4) + (c & 7) * 2; }

// The slots of sequence b begin at cu[b] / 64 + b: ranges of ceil(len / 64) from
// there on never overlap, since floor(x + y) >= floor(x) + floor(y).
__device__ __forceinline__ int64_t first_chunk(int begin, int b) { return begin / kChunk + b; }

// Shared-memory address of the 16-byte vector c of row r in a tile of VECS
// vectors per row, spread so that eight rows of one column hit all banks.
template <int VECS>
__device__ __forceinline__ uint32_t tile_at(uint32_t base, int r, int c) {
    return base + r * (VECS * 16) + ((c ^ (r & (VECS < 8 ? VECS - 1 : 7))) << 4);
}

// Decays are kept in halvings, summed in fp64 and stored as the sum of two floats:
// a difference of two far sums then loses nothing, and 2^x is one instruction.
__device__ __forceinline__ float2 two_floats(double x) {
    const float h = static_cast<float>(x);
    return make_float2(h, static_cast<float>(x - h));
}
__device__ __forceinline__ float decay_between(float2 later, float2 earlier) {
    return exp2f((later.x - earlier.x) + (later.y - earlier.y));
}

// 16x16 fp32 block as a product's operands.  acc + 2^-11 acc_lo += a b.
struct Split4 {
    uint32_t hi[4], lo[4];
};
__device__ __forceinline__ void mma_split(float (&acc)[2][4], float (&acc_lo)[2][4], const Split4& a, const Split4& b) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        mma16816(acc[n], a.hi, b.hi[2 * n], b.hi[2 * n + 1]);
        mma16816(acc_lo[n], a.lo, b.hi[2 * n], b.hi[2 * n + 1]);
        mma16816(acc_lo[n], a.hi, b.lo[2 * n], b.lo[2 * n + 1]);
    }
}
// A result (C fragments of two n8 tiles) as the next product's B operand: 8x8 transposes.
__device__ __forceinline__ void to_b(Split4& b, const float (&x)[2][4]) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            uint32_t hi, lo;
            split_scaled(x[n][e], x[n][e + 1], hi, lo);
            b.hi[2 * n + e / 2] = movm_t(hi);
            b.lo[2 * n + e / 2] = movm_t(lo);
        }
}

// Per chunk and value head.  Q K^T and K K^T by MMA, each warp 16 rows up to the
// diagonal block; then X = (I + A)^-1 by 16x16 blocks: the diagonal ones by
// forward substitution in fp32, one thread a column, the rest
//   X_ij = -X_ii sum_{j <= l < i} A_il X_lj
// by split MMAs, one warp a column of blocks, in registers - the columns do not
// depend on each other - and so P X.
template <int DK>
__global__ void __launch_bounds__(128, 4) chunk_kernel(const DeltaArgs a, Chunk* chunks) {
    constexpr int kVecs = DK / 8;
    extern __shared__ __align__(128) unsigned char smem[];  // K and Q, later the record's image
    // 16x16 blocks, hi and lo, each as four 8x8 matrices in ldmatrix's order for an A operand
    __shared__ __align__(128) __half a_blk[2][6 * 256];     // A below the diagonal blocks
    __shared__ __align__(128) __half p_blk[2][10 * 256];    // P on and below the diagonal
    __shared__ __align__(128) __half x_blk[2][4 * 256];     // inverses of the diagonal blocks
    __shared__ float diag[4][16 * 17];
    __shared__ float4 rows[kChunk];                         // G (two floats), r_k, r_q scale
    __shared__ float bt[kChunk];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.y;
    // the sequence that owns this slot: the last whose first slot is not behind it
    int lo = 0, hi = a.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first_chunk(a.cu[mid], mid) <= blockIdx.x) lo = mid;
        else hi = mid - 1;
    }
    int begin, end, slot;
    if (!sequence(a, lo, begin, end, slot)) return;
    const int64_t local = static_cast<int64_t>(blockIdx.x) - first_chunk(begin, lo);
    if (local < 0 || local * kChunk >= end - begin) return;
    const int t0 = begin + static_cast<int>(local) * kChunk;
    const int n = min(kChunk, end - t0);
    const int kh = h / a.share;

    const uint32_t ks = smem_u32(smem), qs = ks + kChunk * DK * 2;
    {
        constexpr int kStep = 128 / kVecs;
        const int lr = tid / kVecs, lx = tid % kVecs;
        const __half* kp = a.k + static_cast<int64_t>(t0 + lr) * a.k_ts + kh * a.k_hs + lx * 8;
        const __half* qp = a.q + static_cast<int64_t>(t0 + lr) * a.q_ts + kh * a.q_hs + lx * 8;
        const uint32_t dst = tile_at<kVecs>(ks, lr, lx);
#pragma unroll
        for (int i = 0; i < kChunk / kStep; ++i) {
            const bool ok = i * kStep + lr < n;
            cp_async16_or_zero(dst + i * kStep * kVecs * 16, ok ? kp : a.k, ok);
            cp_async16_or_zero(dst + i * kStep * kVecs * 16 + kChunk * DK * 2, ok ? qp : a.q, ok);
            kp += kStep * a.k_ts;
            qp += kStep * a.q_ts;
        }
    }
    cp_async_commit();
    if (warp == 0) {
        // below -200 a decay is 0 in fp32 as it stands, and stays finite here
        double x[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 2 * lane + i;
            const int64_t at = static_cast<int64_t>(t0 + r) * a.v_heads + h;
            const float g = r < n ? a.g[at] : 0.0f;
            x[i] = (g < -200.0f ? -200.0f : g) * 1.4426950408889634074;
            bt[r] = r < n ? a.beta[at] : 0.0f;
        }
        double s = x[0] + x[1];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double u = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += u;
        }
        *reinterpret_cast<float2*>(&rows[2 * lane].x) = two_floats(s - x[1]);
        *reinterpret_cast<float2*>(&rows[2 * lane + 1].x) = two_floats(s);
    }
    cp_async_wait<0>();
    __syncthreads();
    {
        const int r = tid & 63;
        const uint32_t base = tid < 64 ? ks : qs;
        float sum[4] = {};
        if (a.l2_eps >= 0.0f) {
#pragma unroll
            for (int c = 0; c < kVecs; ++c) {
                uint32_t x[4];
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                             : "r"(tile_at<kVecs>(base, r, c)));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = __half22float2(u32_as_h2(x[i]));
                    sum[i] += f.x * f.x + f.y * f.y;
                }
            }
        }
        float norm = a.l2_eps >= 0.0f ? 1.0f / sqrtf((sum[0] + sum[1]) + (sum[2] + sum[3]) + a.l2_eps) : 1.0f;
        if (tid >= 64) norm *= a.scale;
        (tid < 64 ? rows[r].z : rows[r].w) = r < n ? norm : 0.0f;
    }
    __syncthreads();
    Chunk& out = chunks[static_cast<int64_t>(blockIdx.x) * a.v_heads + h];
    if (tid < kChunk) {
        const float4 r = rows[tid], last = rows[kChunk - 1];
        const float eg = exp2f(r.x + r.y);
        out.ck[tid] = eg * r.z;
        out.cq[tid] = eg * r.w;
        out.cs[tid] = decay_between(make_float2(last.x, last.y), make_float2(r.x, r.y)) * r.z;
        if (tid == kChunk - 1) out.keep = eg;
    }

    float kk[8][4], qk[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) kk[j][e] = qk[j][e] = 0.0f;
#pragma unroll
    for (int x = 0; x < DK / 16; ++x) {
        uint32_t ka[4], qa[4];
        const int ar = warp * 16 + (lane & 15), ac = x * 2 + (lane >> 4);
        ldsm4(ka, tile_at<kVecs>(ks, ar, ac));
        ldsm4(qa, tile_at<kVecs>(qs, ar, ac));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > warp) break;
            uint32_t b[4];
            ldsm4(b, tile_at<kVecs>(ks, j * 16 + (lane & 7) + (lane >> 4) * 8, x * 2 + ((lane >> 3) & 1)));
            mma16816(kk[2 * j], ka, b[0], b[1]);
            mma16816(kk[2 * j + 1], ka, b[2], b[3]);
            mma16816(qk[2 * j], qa, b[0], b[1]);
            mma16816(qk[2 * j + 1], qa, b[2], b[3]);
        }
    }
    const int g = lane >> 2, t = lane & 3;
    const float4 row[2] = {rows[warp * 16 + g], rows[warp * 16 + g + 8]};
    const float write[2] = {row[0].z * bt[warp * 16 + g], row[1].z * bt[warp * 16 + g + 8]};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if (j > 2 * warp + 1) break;
        const int c = j * 8 + 2 * t;
        const float4 col[2] = {rows[c], rows[c + 1]};
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
            const int r = warp * 16 + g + e * 4;
            const float4 mine = row[e / 2];
            float p[2], m[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float w = decay_between(make_float2(mine.x, mine.y), make_float2(col[i].x, col[i].y)) * col[i].z;
                p[i] = c + i <= r ? w * mine.w * qk[j][e + i] : 0.0f;
                m[i] = c + i < r ? w * write[e / 2] * kk[j][e + i] : 0.0f;
            }
            // matrices of a block: (rows lo, k lo), (rows hi, k lo), (rows lo, k hi), (rows hi, k hi)
            const int in = ((j & 1) * 2 + e / 2) * 64 + g * 8 + t * 2;
            uint32_t x, y;
            split_scaled(p[0], p[1], x, y);
            const int at = (warp * (warp + 1) / 2 + j / 2) * 256 + in;
            *reinterpret_cast<uint32_t*>(&p_blk[0][at]) = x;
            *reinterpret_cast<uint32_t*>(&p_blk[1][at]) = y;
            if (j / 2 == warp) {
                const int dc = (j & 1) * 8 + 2 * t;
                diag[warp][(g + e * 4) * 17 + dc] = m[0];
                diag[warp][(g + e * 4) * 17 + dc + 1] = m[1];
            } else {
                const int am = (warp * (warp - 1) / 2 + j / 2) * 256 + in;
                split_scaled(m[0], m[1], x, y);
                *reinterpret_cast<uint32_t*>(&a_blk[0][am]) = x;
                *reinterpret_cast<uint32_t*>(&a_blk[1][am]) = y;
            }
        }
    }
    __syncwarp();

    // this warp's diagonal block: lanes 0-15 take a column each,
    // x_i = [i = j] - sum_{l < i} A_il x_l
    float xc[16];
    if (lane < 16) {
        const float* m = diag[warp];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float acc[2] = {i == lane ? 1.0f : 0.0f, 0.0f};
#pragma unroll
            for (int l = 0; l < i; ++l) acc[l & 1] -= m[i * 17 + l] * xc[l];
            xc[i] = acc[0] + acc[1];
            const int at = warp * 256 + ((lane >> 3) * 2 + (i >> 3)) * 64 + (i & 7) * 8 + (lane & 7);
            const __half hi16 = __float2half_rn(xc[i]);
            x_blk[0][at] = hi16;
            x_blk[1][at] = __float2half_rn((xc[i] - __half2float(hi16)) * kLo);
        }
    }
    __syncthreads();     // K and Q are not read any more: the image takes their place

    unsigned char* image = smem;
    constexpr int kImageLo = 128 * kChunk * 2;
    for (int i = tid; i < 6 * 32 * 2 * 2; i += 128) {     // blocks above the diagonal
        const int blk = i / 128, half = (i >> 6) & 1, lo_part = (i >> 5) & 1, r = (i >> 1) & 15, c = i & 1;
        const int bi = blk >= 5 ? 2 : (blk >= 3 ? 1 : 0), bj = blk >= 5 ? 3 : (blk >= 3 ? blk - 1 : blk + 1);
        *reinterpret_cast<uint4*>(image + lo_part * kImageLo + sw128(half * 64 + bi * 16 + r, bj * 16 + c * 8)) =
            make_uint4(0, 0, 0, 0);
    }
    if (lane < 16) {
        const float beta = bt[warp * 16 + lane];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = xc[i] * beta;
            const __half hi16 = __float2half_rn(x);
            const uint32_t at = sw128(warp * 16 + i, warp * 16 + lane);
            *reinterpret_cast<__half*>(image + at) = hi16;
            *reinterpret_cast<__half*>(image + kImageLo + at) = __float2half_rn((x - __half2float(hi16)) * kLo);
        }
    }
    // this warp's column of blocks; its diagonal block as a B operand (k lo, k hi of columns lo, then hi)
    {
        Split4 xb[4];
        const uint32_t xs = smem_u32(x_blk), as = smem_u32(a_blk), ps = smem_u32(p_blk);
        constexpr uint32_t kXLo = 4 * 512, kALo = 6 * 512, kPLo = 10 * 512;
        const float2 beta[2] = {*reinterpret_cast<const float2*>(&bt[warp * 16 + 2 * t]),
                                *reinterpret_cast<const float2*>(&bt[warp * 16 + 8 + 2 * t])};
        auto put_block = [&](int row0, const float (&y)[2][4]) {      // times beta, into columns of this warp
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    uint32_t x, z;
                    split_scaled(y[q][e] * beta[q].x, y[q][e + 1] * beta[q].y, x, z);
                    const uint32_t at = sw128(row0 + g + e * 4, warp * 16 + q * 8 + 2 * t);
                    *reinterpret_cast<uint32_t*>(image + at) = x;
                    *reinterpret_cast<uint32_t*>(image + kImageLo + at) = z;
                }
        };
        ldsm4_t(xb[0].hi, xs + warp * 512 + lane * 16);
        ldsm4_t(xb[0].lo, xs + kXLo + warp * 512 + lane * 16);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int i = warp + s;         // block row
            if (i > 3) break;
            if (s > 0) {
                float y[2][4] = {}, yl[2][4] = {};
#pragma unroll
                for (int l = 0; l < s; ++l) {
                    Split4 m;
                    const uint32_t at = as + (i * (i - 1) / 2 + warp + l) * 512 + lane * 16;
                    ldsm4(m.hi, at);
                    ldsm4(m.lo, at + kALo);
                    mma_split(y, yl, m, xb[l]);
                }
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[q][e] += kLoInv * yl[q][e];
                Split4 yb, m;
                to_b(yb, y);
                ldsm4(m.hi, xs + i * 512 + lane * 16);
                ldsm4(m.lo, xs + kXLo + i * 512 + lane * 16);
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[q][e] = yl[q][e] = 0.0f;
                mma_split(y, yl, m, yb);
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[q][e] = -(y[q][e] + kLoInv * yl[q][e]);
                put_block(i * 16, y);
                to_b(xb[s], y);
            }
            float y[2][4] = {}, yl[2][4] = {};
#pragma unroll
            for (int l = 0; l <= s; ++l) {
                Split4 m;
                const uint32_t at = ps + (i * (i + 1) / 2 + warp + l) * 512 + lane * 16;
                ldsm4(m.hi, at);
                ldsm4(m.lo, at + kPLo);
                mma_split(y, yl, m, xb[l]);
            }
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[q][e] += kLoInv * yl[q][e];
            put_block(64 + i * 16, y);
        }
    }
    __syncthreads();
    uint4* to = reinterpret_cast<uint4*>(out.tp);
#pragma unroll
    for (int i = 0; i < 2 * kImageLo / 16 / 128; ++i) to[i * 128 + tid] = reinterpret_cast<const uint4*>(image)[i * 128 + tid];
}

// The walk, on the tcgen05 tensor cores.  A group of eight warps owns CW value
// columns of a head; a block has NG groups, which share the chunk's tiles, and four
// warps that load them ahead.  Per chunk and group three products, each with M =
// 128 rows and N = 2 CW columns (the hi and the lo half of a split operand side by
// side, so that the other operand is read once for both):
//   D1 = [K; Q] S0        rows 0-63 give R = V - diag(ck) K S0, rows 64-127 the outputs' first part
//   D2 = [T; P T] R       rows 0-63 give U, rows 64-127 the outputs' second part
//   D3 = K^T diag(cs) U   the state's new part; K's tile serves as its own transpose (M-major operand)
// A row of a product belongs to one thread of each of the group's two
// warpgroups (half of the columns each), so every scale is a thread's own and the
// state stays in registers, CW / 2 values per thread.  Between products only R, U
// or S goes through shared memory, in the layout of the next B operand.
//
// A walk's speed is this chain, not its operations: three times issue, MMA (about
// 32 clocks per 16 of K, the reading of the 128-row operand) and a pass over the
// accumulator.  So a small call takes CW = 16 (most blocks), a large one two groups
// of 32 columns per block, whose chains interleave on one tensor core.
template <int DK, int CW, int NG>
struct Walk {
    static constexpr int kThreads = NG * 256 + 128;
    static constexpr int kSub = DK / 64;                   // 64 columns of K, Q: one 128-byte tile
    static constexpr int kTile = 128 * 128;                // 128 rows of 128 bytes
    static constexpr int kRec = kSub * kTile;              // offset of the chunk's record in a stage
    static constexpr int kVRow = NG * CW * 2;
    static constexpr int kV = kRec + sizeof(Chunk);
    static constexpr int kStage = (kV + kChunk * kVRow + 1023) / 1024 * 1024;
    static constexpr int kBTile = 2 * CW * 128;            // a B operand with K = 64
    static constexpr int kGroup = (kSub + 1) * kBTile;     // S, then R and U in turn
    static constexpr int kStages = NG * CW == 16 ? 3 : 2;
    static constexpr int kSmem = kStages * kStage + NG * kGroup + 1024;
    static constexpr int kAcc = 2 * CW;                    // tensor-memory columns of an accumulator
    static constexpr int kTmem = NG * 3 * kAcc <= 128 ? 128 : (NG * 3 * kAcc <= 256 ? 256 : 512);
    static_assert(kSmem <= 232448 - 256, "shared memory");
};

// CT consecutive fp32 columns of this warp's 32 lanes.
template <int CT>
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[CT]) {
    static_assert(CT == 8 || CT == 16, "");
    uint32_t r[CT];
    if constexpr (CT == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(addr));
    else
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(addr));
#pragma unroll
    for (int i = 0; i < CT; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

template <int DK, int CW, int NG>
__global__ void __launch_bounds__(NG * 256 + 128, 1) walk_kernel(const DeltaArgs a, const Chunk* chunks) {
    using C = Walk<DK, CW, NG>;
    constexpr int kVecs = DK / 8;
    constexpr int CT = CW / 2;        // columns of a thread
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages], made[NG];
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, lane = tid & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
    if (tid < 32) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(C::kTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 32) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&full[i], 129);      // the loading threads, and the announcement of the bulk copy
            mbar_init(&empty[i], NG);
        }
        for (int i = 0; i < NG; ++i) mbar_init(&made[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_trigger();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();

    const int h = blockIdx.y, b = blockIdx.z;
    const int col0 = blockIdx.x * NG * CW;
    int begin = 0, end = 0, slot = 0;
    const bool valid = sequence(a, b, begin, end, slot);
    const int chunks_here = valid ? (end - begin + kChunk - 1) / kChunk : 0;
    // Every wait is bounded.  A thread whose wait gave up records it and goes on
    // without waiting, so that all barriers still meet and the block ends.
    bool dead = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!dead && !mbar_wait(bar, parity)) {
            dead = true;
            atomicOr(&g_gated_delta_dev_error, kDevErrTimeout);
        }
    };
    auto arrive = [](uint64_t* bar) {
        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
    };

    if (tid >= NG * 256) {
        // ---- the loading warps ----
        constexpr int kStep = 128 / kVecs;           // rows of one sweep of the 128 threads; a multiple of 8,
        static_assert(kStep % 8 == 0, "swizzle");    // so a thread keeps its place in the swizzle
        const int kh = h / a.share, lt = tid - NG * 256;
        const int lr = lt / kVecs, lx = lt % kVecs;
        const __half* kp = a.k + static_cast<int64_t>(begin + lr) * a.k_ts + kh * a.k_hs + lx * 8;
        const __half* qp = a.q + static_cast<int64_t>(begin + lr) * a.q_ts + kh * a.q_hs + lx * 8;
        const int64_t k_step = kStep * a.k_ts, q_step = kStep * a.q_ts;
        const Chunk* rec = chunks + first_chunk(begin, b) * a.v_heads + h;
        for (int c = 0; c < chunks_here; ++c) {
            const int st = c % C::kStages;
            if (c >= C::kStages) wait(&empty[st], (c / C::kStages - 1) & 1);
            const uint32_t stage = base + st * C::kStage;
            if (lt == 0) {
                mbar_expect_tx(&full[st], sizeof(Chunk));
                bulk_load(smem + st * C::kStage + C::kRec, rec, sizeof(Chunk), &full[st]);
            }
            rec += a.v_heads;
            const uint32_t dst = stage + (lx >> 3) * C::kTile + sw128(lr, (lx & 7) * 8);
            const int t0 = begin + c * kChunk;
            const int n = min(kChunk, end - t0);
#pragma unroll
            for (int i = 0; i < kChunk / kStep; ++i) {
                const bool ok = i * kStep + lr < n;
                cp_async16_or_zero(dst + i * kStep * 128, ok ? kp : a.k, ok);
                cp_async16_or_zero(dst + (kChunk + i * kStep) * 128, ok ? qp : a.q, ok);
                kp += k_step;
                qp += q_step;
            }
            constexpr int kVV = NG * CW / 8;      // 16-byte vectors of a row of V
#pragma unroll
            for (int i = 0; i < kChunk * kVV / 128; ++i) {
                const int item = i * 128 + lt, r = item / kVV, x = item % kVV;
                const bool ok = r < n && col0 + x * 8 < a.dv;
                cp_async16_or_zero(tile_at<kVV>(stage + C::kV, r, x),
                                   ok ? a.v + static_cast<int64_t>(t0 + r) * a.v_ts + h * a.v_hs + col0 + x * 8 : a.v, ok);
            }
            cp_async_commit();
            cp_async_wait<0>();
            fence_proxy_async_smem();      // the MMAs read through the async proxy
            arrive(&full[st]);
        }
        // bulk copies land before the block's shared memory goes
        if (lt == 0)
            for (int c = max(0, chunks_here - C::kStages); c < chunks_here; ++c) wait(&full[c % C::kStages], (c / C::kStages) & 1);
    } else {
        const int group = tid >> 8, gt = tid & 255, half = gt >> 7, quarter = (tid >> 5) & 3;
        const int row = quarter * 32 + lane;          // of every product
        const int tok = row & 63;
        const bool state_row = quarter < 2;           // of D1 and D2: a token's state part, or its output part
        const int colg = group * CW + half * CT;      // first column of this thread within the block
        const int col = col0 + colg;
        const bool live = col < a.dv;                 // value_dim is a multiple of 16: CT columns are in or out together
        const uint32_t bt = base + C::kStages * C::kStage + group * C::kGroup, rt = bt + C::kSub * C::kBTile;
        const uint32_t acc = tmem + group * 3 * C::kAcc;
        const uint32_t acc_lane = acc + (static_cast<uint32_t>(quarter * 32) << 16) + half * CT;
        auto rows_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + 2 * group) : "memory"); };
        auto group_sync = [&]() { asm volatile("bar.sync %0, 256;" ::"r"(2 + 2 * group) : "memory"); };
        // a split value as element k of rows n (hi) and CW + n (lo) of a B tile
        auto put = [&](uint32_t tile, int n, int k, float x) {
            const __half hi = __float2half_rn(x);
            const __half lo = __float2half_rn((x - __half2float(hi)) * kLo);
            const uint32_t at = tile + sw128(n, k);
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(__half_as_ushort(hi)) : "memory");
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + CW * 128), "h"(__half_as_ushort(lo)) : "memory");
        };
        // a product's hi + 2^-11 lo for this thread's row and columns
        auto take = [&](int d, float (&x)[CT]) {
            float lo[CT];
            tmem_ld<CT>(acc_lane + d * C::kAcc, x);
            tmem_ld<CT>(acc_lane + d * C::kAcc + CW, lo);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < CT; ++i) x[i] += kLoInv * lo[i];
        };

        // this thread's row of the state
        float s[CT];
        const int64_t at = ((static_cast<int64_t>(slot) * a.v_heads + h) * DK + row) * a.dv + col;
        const bool has_state = row < DK && live && valid;
#pragma unroll
        for (int i = 0; i < CT; i += 4) {
            const float4 x = a.state_in && has_state ? *reinterpret_cast<const float4*>(a.state_in + at + i)
                                                     : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            s[i] = x.x, s[i + 1] = x.y, s[i + 2] = x.z, s[i + 3] = x.w;
        }
        auto put_state = [&]() {
            if (row < DK) {
#pragma unroll
                for (int i = 0; i < CT; ++i) put(bt + (row >> 6) * C::kBTile, half * CT + i, row & 63, s[i]);
            }
            fence_proxy_async_smem();
            tc_fence_before();
            group_sync();
        };
        put_state();

        constexpr uint32_t kWide = instr_desc_f16(128, 2 * CW), kNarrow = instr_desc_f16(128, CW);
        constexpr uint32_t kMajorM = kWide | (1u << 15);      // A stored with M contiguous
        uint32_t phase = 0;
        for (int c = 0; c < chunks_here; ++c) {
            const int st = c % C::kStages;
            const uint32_t stage = base + st * C::kStage;
            const float* scales = reinterpret_cast<const float*>(smem + st * C::kStage + C::kRec + sizeof(__half) * 2 * 128 * kChunk);
            wait(&full[st], (c / C::kStages) & 1);
            if (gt == 0) {
                tc_fence_after();
#pragma unroll
                for (int j = 0; j < DK / 16; ++j)
                    mma_f16_ss(acc, smem_desc_sw128(stage + (j / 4) * C::kTile + (j % 4) * 32),
                               smem_desc_sw128(bt + (j / 4) * C::kBTile + (j % 4) * 32), kWide, j > 0);
                mma_commit(&made[group]);
            }
            __syncwarp();
            // what the pass over D1 needs, while the MMAs run
            const float scale = scales[(state_row ? 0 : kChunk) + tok], cs = scales[2 * kChunk + tok], keep = scales[3 * kChunk];
            uint4 vv[CT / 8];
#pragma unroll
            for (int i = 0; i < CT / 8; ++i)
                vv[i] = *reinterpret_cast<const uint4*>(smem + (tile_at<NG * CW / 8>(stage + C::kV, tok, colg / 8 + i) - base));
            wait(&made[group], phase);
            phase ^= 1;
            __syncwarp();
            tc_fence_after();
            float x[CT], o[CT];
            take(0, x);
            tc_fence_before();
            if (state_row) {
#pragma unroll
                for (int i = 0; i < CT; i += 2) {
                    const float2 v = __half22float2(u32_as_h2((&vv[i / 8].x)[(i & 7) / 2]));
                    put(rt, half * CT + i, tok, v.x - scale * x[i]);
                    put(rt, half * CT + i + 1, tok, v.y - scale * x[i + 1]);
                }
                fence_proxy_async_smem();
                rows_sync();
                if (gt == 0) {
                    tc_fence_after();
                    const uint32_t tp = stage + C::kRec;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint64_t r = smem_desc_sw128(rt + j * 32);
                        mma_f16_ss(acc + C::kAcc, smem_desc_sw128(tp + j * 32), r, kWide, j > 0);
                        mma_f16_ss(acc + C::kAcc + CW, smem_desc_sw128(tp + C::kTile + j * 32), r, kNarrow, 1);
                    }
                    mma_commit(&made[group]);
                }
                __syncwarp();
            } else {
#pragma unroll
                for (int i = 0; i < CT; ++i) o[i] = scale * x[i];
            }
            wait(&made[group], phase);
            phase ^= 1;
            __syncwarp();
            tc_fence_after();
            take(1, x);
            tc_fence_before();
            if (state_row) {
#pragma unroll
                for (int i = 0; i < CT; ++i) put(rt, half * CT + i, tok, cs * x[i]);
                fence_proxy_async_smem();
                rows_sync();
                if (gt == 0) {
                    tc_fence_after();
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        // K^T: blocks of 64 rows lie a tile apart (with 64 of them, the second block is Q's, its
                        // results unused), groups of 8 tokens 1024 bytes
                        const uint64_t kt = (smem_desc_sw128(stage + j * 2048) & ~(static_cast<uint64_t>(0x3fff) << 16)) |
                                            (static_cast<uint64_t>((C::kSub == 2 ? C::kTile : 8192) >> 4) << 16);
                        mma_f16_ss(acc + 2 * C::kAcc, kt, smem_desc_sw128(rt + j * 32), kMajorM, j > 0);
                    }
                    mma_commit(&made[group]);
                }
                __syncwarp();
            } else {
                const int token = begin + c * kChunk + tok;
                if (live && token < end) {
                    uint32_t r[CT / 2];
#pragma unroll
                    for (int i = 0; i < CT; i += 2) r[i / 2] = h2_as_u32(__floats2half2_rn(o[i] + x[i], o[i + 1] + x[i + 1]));
                    uint4* to = reinterpret_cast<uint4*>(a.out + (static_cast<int64_t>(token) * a.v_heads + h) * a.dv + col);
#pragma unroll
                    for (int i = 0; i < CT / 8; ++i) to[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                }
            }
            wait(&made[group], phase);
            phase ^= 1;
            __syncwarp();
            tc_fence_after();
            take(2, x);
#pragma unroll
            for (int i = 0; i < CT; ++i) s[i] = keep * s[i] + x[i];
            put_state();
            if (gt == 0) arrive(&empty[st]);
        }
        if (a.state_out && has_state) {
#pragma unroll
            for (int i = 0; i < CT; i += 4)
                *reinterpret_cast<float4*>(a.state_out + at + i) = make_float4(s[i], s[i + 1], s[i + 2], s[i + 3]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid < 32)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmem) : "memory");
}

int64_t chunk_slots(int64_t tokens, int64_t batch) { return tokens / kChunk + batch; }

template <int DK, int CW, int NG>
int launch_walk(const DeltaArgs& a, const Chunk* chunks, cudaStream_t stream) {
    using C = Walk<DK, CW, NG>;
    static std::atomic<uint64_t> done{0};
    const int st = allow_smem(walk_kernel<DK, CW, NG>, C::kSmem, done);
    if (st) return st;
    return launch(walk_kernel<DK, CW, NG>, dim3((a.dv + NG * CW - 1) / (NG * CW), a.v_heads, a.batch), dim3(C::kThreads),
                  C::kSmem, stream, a, chunks);
}

template <int DK>
int run_chunked(const DeltaArgs& a, void* workspace, cudaStream_t stream) {
    Chunk* chunks = static_cast<Chunk*>(workspace);
    constexpr int kSmem = 32768;      // K and Q (at most 64 rows of 256 bytes each), then the record's image
    static std::atomic<uint64_t> done{0};
    int st = allow_smem(chunk_kernel<DK>, kSmem, done);
    if (st) return st;
    st = launch(chunk_kernel<DK>, dim3(static_cast<unsigned>(chunk_slots(a.tokens, a.batch)), a.v_heads), dim3(128),
                kSmem, stream, a, chunks);
    if (st) return st;
    // the narrowest blocks that still all run at once
    const int64_t heads = static_cast<int64_t>(a.batch) * a.v_heads;
    if (heads * ((a.dv + 15) / 16) <= sm_count()) return launch_walk<DK, 16, 1>(a, chunks, stream);
    if (heads * ((a.dv + 31) / 32) <= sm_count()) return launch_walk<DK, 32, 1>(a, chunks, stream);
    return launch_walk<DK, 32, 2>(a, chunks, stream);
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
    return static_cast<size_t>(chunk_slots(tokens, batch)) * v_heads * sizeof(Chunk);
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
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return args->key_dim == 128 ? run_chunked<128>(a, workspace, s) : run_chunked<64>(a, workspace, s);
}

}  // extern "C"
