// The gated delta rule of the linear-attention layers.  Per value head, with a
// state S [Dk][Dv] (fp32) and per token q, k (Dk), v (Dv), a log decay g and a
// write strength beta:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q,
// with q and k divided by sqrt(sum x^2 + eps) first when asked.  Value heads
// h * v_heads / k_heads ... share key head h.
#include "mixing.cuh"
#include "tcgen05.cuh"

#include <cmath>
#include <type_traits>

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
    const int32_t* cu;        // prompts: sequence b has tokens cu[b] .. cu[b + 1] - 1
    int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs;
    int batch, tokens, slots, v_heads, share, dv;
    float scale, l2_eps;
};

// The tokens and the state slot of sequence b; false: nothing to do.
__device__ __forceinline__ bool sequence(const DeltaArgs& a, int b, int& begin, int& end, int& slot) {
    slot = a.index ? a.index[b] : b;
    begin = a.cu[b];
    end = a.cu[b + 1];
    if (slot < 0) return false;
    if (slot >= a.slots || begin < 0 || end < begin || end > a.tokens) {
        if (threadIdx.x == 0) atomicOr(&g_gated_delta_dev_error, kDevErrIndex);
        return false;
    }
    return true;
}

// ---- one token per sequence -----------------------------------------------------
//
// Bound by the state's bytes (8 Dk Dv per head, read and written once; 7 operations
// per element).  A warp keeps 16 columns of a head's state in registers - 8 lane
// groups take every eighth row, four lanes a 64-byte row piece - and works
// without any block-wide step: the products S^T k and S^T q are taken in one
// pass over the old state, since S_new^T q = e^g S^T q + (k.q) u.
constexpr int kCols = 16;
constexpr int kStepWarps = 2;

template <int DK>
__global__ void __launch_bounds__(kStepWarps * 32) step_kernel(const DeltaArgs a) {
    constexpr int kRows = DK / 8;    // rows of a lane
    constexpr int kPer = DK / 32;    // q, k elements of a lane
    __shared__ float2 kq[kStepWarps][DK];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int col = (blockIdx.x * (blockDim.x >> 5) + warp) * kCols + (lane & 3) * 4;
    const int rg = lane >> 2;
    const int64_t b = blockIdx.z;
    const int h = blockIdx.y, slot = a.index ? a.index[b] : static_cast<int>(b);
    if (slot < 0 || col >= a.dv) return;
    if (slot >= a.slots) {
        if (threadIdx.x == 0) atomicOr(&g_gated_delta_dev_error, kDevErrIndex);
        return;
    }
    const int64_t at = ((static_cast<int64_t>(slot) * a.v_heads + h) * DK + rg) * a.dv + col;
    float4 s[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) s[i] = *reinterpret_cast<const float4*>(a.state_in + at + static_cast<int64_t>(i) * 8 * a.dv);
    const int kh = h / a.share;
    const __half* qp = a.q + b * a.q_ts + kh * a.q_hs + lane * kPer;
    const __half* kp = a.k + b * a.k_ts + kh * a.k_hs + lane * kPer;
    const uint2 vv = *reinterpret_cast<const uint2*>(a.v + b * a.v_ts + h * a.v_hs + col);
    const float decay = expf(a.g[b * a.v_heads + h]), beta = a.beta[b * a.v_heads + h];
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
        *reinterpret_cast<float4*>(a.state_out + at + static_cast<int64_t>(i) * 8 * a.dv) = s[i];
    }
    if (rg == 0)
        *reinterpret_cast<uint2*>(a.out + (b * a.v_heads + h) * a.dv + col) =
            make_uint2(h2_as_u32(__floats2half2_rn(o[0], o[1])), h2_as_u32(__floats2half2_rn(o[2], o[3])));
}

int run_step(const DeltaArgs& a, int dk, cudaStream_t stream) {
    // Two warps a block (one while that leaves SMs without a block): a block's registers are only free for the
    // next when its last warp ends, and with eight warps a block 160 sequences of 32 heads took 114 us instead of
    // 99 (654 MB, 100 at the copy rate).
    const int cols = a.dv / kCols;
    int warps = cols > 1 ? kStepWarps : 1;
    if (static_cast<int64_t>(a.batch) * a.v_heads * ((cols + warps - 1) / warps) < 2 * sm_count()) warps = 1;
    const dim3 grid((cols + warps - 1) / warps, a.v_heads, a.batch);
    return launch(dk == 128 ? step_kernel<128> : step_kernel<64>, grid, dim3(warps * 32), 0, stream, a);
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
// a single fp16 operand would leave 2^-11.  T, P T and the blocks that they are made
// from are bounded and kept times 2^13 and 2^12, for they meet the largest values: a
// decayed element of 2^-20 has its 22 bits too.  (State values and written rows are
// below fp16's 65504 then; with |k| <= 1, beta <= 2 and g <= 0 they are bounded by
// the state's start and twice the sum of |v|.)
constexpr int kChunk = 64;
constexpr int kLoBits = 11;
constexpr float kLo = 2048.0f, kLoInv = 1.0f / 2048.0f;      // 2^kLoBits

// x *= a, y *= b in one instruction.
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b) {
    asm("{\n\t.reg .b64 v, f;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 f, {%2, %3};\n\tmul.rn.f32x2 v, v, f;\n\tmov.b64 {%0, %1}, v;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}
__device__ __forceinline__ void split_scaled(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = h2_as_u32(__floats2half2_rn(x, y));
    mul2(x, y, kLo, kLo);
    fma2_f16_f32(x, y, hi, 0xe800e800u);      // - 2^11 hi: exact
    lo = h2_as_u32(__floats2half2_rn(x, y));
}

// One chunk's share of the workspace: T and P T (its rows for q of norm 1 or less),
// both at most 4 in magnitude (1 with beta <= 1) and kept times 2^13 as hi + 2^-11 lo, and the scales.  Of the
// two matrices only the 16x16 blocks on and below the diagonal are kept, block column
// after block column, each block as four 8x8 matrices of 128 contiguous bytes:
// fragments are written and read whole, ldmatrix hits no bank twice, a block
// column is an MMA's operand of 64 - 16 j rows, and a chunk is one copy.
constexpr int kTri = 40 * 64;        // elements of a triangle
constexpr float kTriScale = 8192.0f;
constexpr float kBlockScale = 4096.0f;      // of the chunk kernel's blocks: A, P, X and A X are at most 2 in magnitude
struct Chunk {
    __half tp[2][2][kTri];           // [hi, lo][T, P T]
    float ck[kChunk];                // e^G r_k
    float cq[kChunk];                // scale e^G r_q
    float cs[kChunk];                // e^(G_C - G) r_k 2^-13
    float oq[kChunk];                // scale r_q |q's row in P T|^-1 2^-13
    float keep;                      // e^G_C
    float pad[63];
};
static_assert(sizeof(Chunk) % 128 == 0, "chunks stay aligned");
constexpr uint32_t kTriBytes = 4 * kTri * 2, kScaleBytes = (4 * kChunk + 4) * 4;
constexpr uint32_t kChunkBytes = kTriBytes + kScaleBytes;      // in use
// Block (i, j) of a triangle, in blocks of 512 bytes; i counts on from column j's start.
__host__ __device__ constexpr int tri_column(int j) { return j * (9 - j) / 2; }
__host__ __device__ constexpr int tri_block(int i, int j) { return tri_column(j) + i - j; }

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
__device__ __forceinline__ float pow2(float x) {       // below 2^-126: 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float decay_between(float2 later, float2 earlier) {
    return pow2((later.x - earlier.x) + (later.y - earlier.y));
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
// Per chunk and value head, four warps.
//
// Q K^T and K K^T by MMA in 16x16 blocks on and below the diagonal, three or two
// per warp, one of them on the diagonal.  Below it a decay e^(G_r - G_c) is split at
// the row block's start into a factor of the row and one of the column, neither
// above 1 where g <= 0, so that an element costs a product and not an exponential.
//
// Then X = (I + A)^-1: the diagonal blocks by forward substitution in fp32, one
// thread a column; the others by split MMAs (operands hi + 2^-11 lo), first
// X_10 and X_32, then the lower left quarter -X_B (A_BA X_A), so that no warp
// waits for more than four steps; and P X beside and behind them.
//
// 8256 chunks of 64 tokens (16 heads of 128, 409 MB with what stays in L2): 143 us, 2.6 us a chunk and
// SM, where the copy rate would take 67.  Bound by its instructions and shared memory: 9200 warp
// instructions a chunk, issued in 54 % of the cycles, shared memory busy in 67 %, DRAM in 37 %
// (152 us before the triangle's blocks were dealt out evenly, 262 with a warp a block row).
template <int DK>
struct ChunkSmem {
    static constexpr int kKQ = 2 * kChunk * DK * 2;
    static constexpr int kA = 0, kP = kA + 6 * 1024, kX = kP + 10 * 1024, kY = kX + 10 * 1024, kDiag = kY + 4 * 1024;
    static constexpr int kDiagRow = 20;                    // floats
    static constexpr int kWork = kDiag + 4 * 16 * kDiagRow * 4;
    static constexpr int kBytes = kKQ > kWork ? kKQ : kWork;
};

template <int DK>
__global__ void __launch_bounds__(128, 5) chunk_kernel(const DeltaArgs a, Chunk* chunks) {
    using M = ChunkSmem<DK>;
    constexpr int kVecs = DK / 8;
    // K and Q; then blocks of 16x16, hi and lo of 512 bytes, each as four 8x8 matrices in ldmatrix's order for
    // an A operand: (rows lo, k lo), (rows hi, k lo), (rows lo, k hi), (rows hi, k hi)
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float4 rows[kChunk];                         // G (two floats), r_k, r of q's row
    __shared__ float2 row_by[kChunk];                       // factors of a row below the diagonal: of A, of P
    __shared__ float col_by[96];                            // factors of columns 0 .. 16 i - 1 for row block i = 1, 2, 3
    __shared__ float bt[kChunk], qn[kChunk];                // beta; scale of an output over that of q's row
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

    const uint32_t base = smem_u32(smem), ks = base, qs = ks + kChunk * DK * 2;
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
        const uint32_t from = tid < 64 ? ks : qs;
        float sum[4] = {};
        if (a.l2_eps >= 0.0f || tid >= 64) {
#pragma unroll
            for (int c = 0; c < kVecs; ++c) {
                uint32_t x[4];
                asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                             : "r"(tile_at<kVecs>(from, r, c)));
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = __half22float2(u32_as_h2(x[i]));
                    sum[i] += f.x * f.x + f.y * f.y;
                }
            }
        }
        const float square = (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (tid < 64) {
            rows[r].z = r < n ? (a.l2_eps >= 0.0f ? 1.0f / sqrtf(square + a.l2_eps) : 1.0f) : 0.0f;
        } else {
            // P's rows are made for q of norm 1 or less, whether or not q is to be normalised
            const float norm = a.l2_eps >= 0.0f ? sqrtf(square + a.l2_eps) : (square > 0.0f ? sqrtf(square) : 1.0f);
            rows[r].w = r < n ? 1.0f / norm : 0.0f;
            qn[r] = a.scale * (a.l2_eps >= 0.0f ? 1.0f : norm);
        }
    }
    __syncthreads();
    Chunk& out = chunks[static_cast<int64_t>(blockIdx.x) * a.v_heads + h];
    auto g_at = [&](int r) { return *reinterpret_cast<const float2*>(&rows[r].x); };
    if (tid < kChunk) {
        const float4 r = rows[tid];
        const float eg = pow2(r.x + r.y);
        out.ck[tid] = eg * r.z;
        out.cq[tid] = eg * r.w * qn[tid];
        out.cs[tid] = decay_between(g_at(kChunk - 1), make_float2(r.x, r.y)) * r.z * (1.0f / kTriScale);
        out.oq[tid] = qn[tid] * (1.0f / kTriScale);
        if (tid == kChunk - 1) out.keep = eg;
        if (tid >= 16) {
            const float f = decay_between(make_float2(r.x, r.y), g_at((tid & ~15) - 1));
            row_by[tid] = make_float2(f * r.z * bt[tid] * kBlockScale, f * r.w * kBlockScale);
        }
    }
    if (tid >= 32) {
        const int i = tid - 32;
        const int block = i < 16 ? 1 : (i < 48 ? 2 : 3), c = i - (block == 1 ? 0 : (block == 2 ? 16 : 48));
        col_by[i] = decay_between(g_at(block * 16 - 1), g_at(c)) * rows[c].z;
    }

    // this warp's blocks: two in one row of blocks, and with warps 0 and 2 a third; the last on the diagonal
    const int row01 = warp == 0 ? 3 : (warp == 1 ? 3 : (warp == 2 ? 2 : 1)), col0 = warp == 1 ? 2 : 0;
    const bool third = !(warp & 1);
    const int own = warp == 0 ? 0 : 4 - warp;         // its diagonal block: 0, 3, 2, 1
    float kk[3][2][4], qk[3][2][4];
#pragma unroll
    for (int j = 0; j < 3; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) kk[j][e >> 2][e & 3] = qk[j][e >> 2][e & 3] = 0.0f;
    const int a_row = lane & 15, a_vec = lane >> 4, b_row = (lane & 7) + (lane >> 4) * 8, b_vec = (lane >> 3) & 1;
#pragma unroll
    for (int x = 0; x < DK / 16; ++x) {
        uint32_t ka[4], qa[4], b[4];
        ldsm4(ka, tile_at<kVecs>(ks, row01 * 16 + a_row, x * 2 + a_vec));
        ldsm4(qa, tile_at<kVecs>(qs, row01 * 16 + a_row, x * 2 + a_vec));
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            if (j == 2) {
                if (!third) break;
                if (warp == 0) {
                    ldsm4(ka, tile_at<kVecs>(ks, a_row, x * 2 + a_vec));
                    ldsm4(qa, tile_at<kVecs>(qs, a_row, x * 2 + a_vec));
                }
            }
            ldsm4(b, tile_at<kVecs>(ks, (j < 2 ? col0 + j : own) * 16 + b_row, x * 2 + b_vec));
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                mma16816(kk[j][q], ka, b[2 * q], b[2 * q + 1]);
                mma16816(qk[j][q], qa, b[2 * q], b[2 * q + 1]);
            }
        }
    }
    __syncthreads();     // K and Q are not read any more
    const int g = lane >> 2, t = lane & 3;
    // values of an accumulator as block `to` in shared memory
    auto put = [&](int to, const float (&x)[2][4]) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                uint32_t u, l;
                split_scaled(x[q][e], x[q][e + 1], u, l);
                uint32_t* at = reinterpret_cast<uint32_t*>(smem + to + (q * 2 + e / 2) * 128 + g * 16 + t * 4);
                at[0] = u;
                at[128] = l;
            }
    };
    auto tri = [](int i, int j) { return (i * (i + 1) / 2 + j) * 1024; };      // of P and X
    auto below = [](int i, int j) { return (i * (i - 1) / 2 + j) * 1024; };    // of A
    float* diag = reinterpret_cast<float*>(smem + M::kDiag) + own * 16 * M::kDiagRow;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        if (j == 2 && !third) break;
        const int bi = j < 2 ? row01 : own, bj = j < 2 ? col0 + j : own;
        if (bi != bj) {
            const float* cb = col_by + (bi == 1 ? 0 : (bi == 2 ? 16 : 48)) + bj * 16 + 2 * t;
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float2 rb = row_by[bi * 16 + g + e * 4];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const float2 c = *reinterpret_cast<const float2*>(cb + q * 8);
                    kk[j][q][e] *= rb.x * c.x, kk[j][q][e + 1] *= rb.x * c.y;
                    qk[j][q][e] *= rb.y * c.x, qk[j][q][e + 1] *= rb.y * c.y;
                }
            }
            put(M::kA + below(bi, bj), kk[j]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const int r = g + e * 4;
                const float4 mine = rows[bi * 16 + r];
                const float write = mine.z * bt[bi * 16 + r];
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int c = q * 8 + 2 * t + i;
                        const float4 col = rows[bi * 16 + c];
                        const float w = decay_between(make_float2(mine.x, mine.y), make_float2(col.x, col.y)) * col.z;
                        diag[r * M::kDiagRow + c] = c < r ? w * write * kk[j][q][e + i] : 0.0f;
                        qk[j][q][e + i] = c <= r ? w * (mine.w * kBlockScale) * qk[j][q][e + i] : 0.0f;
                    }
            }
        }
        put(M::kP + tri(bi, bj), qk[j]);
    }
    __syncwarp();

    // the diagonal block: lanes 0-15 take a column each, x_i = [i = j] - sum_{l < i} A_il x_l
    if (lane < 16) {
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float acc[4] = {i == lane ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int l = 0; l < i; l += 4) {
                const float4 m = *reinterpret_cast<const float4*>(diag + i * M::kDiagRow + l);     // zeros from l = i on
                acc[0] -= m.x * x[l];
                if (l + 1 < i) acc[1] -= m.y * x[l + 1];
                if (l + 2 < i) acc[2] -= m.z * x[l + 2];
                if (l + 3 < i) acc[3] -= m.w * x[l + 3];
            }
            x[i] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
        }
        __syncwarp(0xffffu);      // all of A's block has been read
#pragma unroll
        for (int i = 0; i < 16; ++i) diag[i * M::kDiagRow + lane] = x[i];
    }
    __syncwarp();

    float y[2][4], yl[2][4];
    auto start = [&]() {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[q][e] = yl[q][e] = 0.0f;
    };
    // (y, yl) += block at `left` times block at `right`; finish leaves y in the blocks' scale
    auto times = [&](int left, int right) {
        Split4 l, r;
        ldsm4(l.hi, base + left + lane * 16);
        ldsm4(l.lo, base + left + 512 + lane * 16);
        ldsm4_t(r.hi, base + right + lane * 16);
        ldsm4_t(r.lo, base + right + 512 + lane * 16);
        mma_split(y, yl, l, r);
    };
    auto finish = [&](float sign) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[q][e] = (sign / kBlockScale) * (y[q][e] + kLoInv * yl[q][e]);
    };
    // y times beta (2^13 in all) as block (i, j) of the record's T (0) or P T (1)
    auto record = [&](int which, int i, int j) {
        const int in = tri_block(i, j) * 256 + g * 8 + t * 2;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const float2 b = *reinterpret_cast<const float2*>(&bt[j * 16 + q * 8 + 2 * t]);
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                uint32_t u, l;
                split_scaled(y[q][e] * (b.x * (kTriScale / kBlockScale)), y[q][e + 1] * (b.y * (kTriScale / kBlockScale)), u, l);
                const int at = in + (e / 2) * 128 + q * 64;
                *reinterpret_cast<uint32_t*>(&out.tp[0][which][at]) = u;
                *reinterpret_cast<uint32_t*>(&out.tp[1][which][at]) = l;
            }
        }
    };
    auto put_x = [&](int i, int j) {
        put(M::kX + tri(i, j), y);
        record(0, i, j);
    };
    auto p_times = [&](int i, int j) {
        start();
#pragma unroll 1
        for (int l = j; l <= i; ++l) times(M::kP + tri(i, l), M::kX + tri(l, j));
        finish(1.0f);
        record(1, i, j);
    };
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[q][e] = kBlockScale * diag[(g + (e >> 1) * 8) * M::kDiagRow + q * 8 + 2 * t + (e & 1)];
    put_x(own, own);
    __syncthreads();
    auto y_at = [](int i, int j) { return M::kY + ((i - 2) * 2 + j) * 1024; };
    if (warp < 2) {          // X_10, X_32; the products go through shared memory of Y_20, Y_30
        const int i = warp == 0 ? 1 : 3, j = i - 1;
        start();
        times(M::kA + below(i, j), M::kX + tri(j, j));
        finish(1.0f);
        put(y_at(2 + warp, 0), y);
        __syncwarp();
        start();
        times(M::kX + tri(i, i), y_at(2 + warp, 0));
        finish(-1.0f);
        put_x(i, j);
    } else {                 // Y_21, Y_31
        start();
        times(M::kA + below(warp, 1), M::kX + tri(1, 1));
        finish(1.0f);
        put(y_at(warp, 1), y);
    }
    __syncthreads();
    if (warp < 2) {          // Y_20, Y_30
        start();
        times(M::kA + below(2 + warp, 0), M::kX + tri(0, 0));
        times(M::kA + below(2 + warp, 1), M::kX + tri(1, 0));
        finish(1.0f);
        put(y_at(2 + warp, 0), y);
    } else {                 // X_21, X_31
        start();
        if (warp == 3) times(M::kX + tri(3, 2), y_at(2, 1));
        times(M::kX + tri(warp, warp), y_at(warp, 1));
        finish(-1.0f);
        put_x(warp, 1);
    }
    __syncthreads();
    if (warp < 2) {          // X_20, X_30
        start();
        if (warp == 1) times(M::kX + tri(3, 2), y_at(2, 0));
        times(M::kX + tri(2 + warp, 2 + warp), y_at(2 + warp, 0));
        finish(-1.0f);
        put_x(2 + warp, 0);
    } else if (warp == 2) {
        p_times(3, 1);
        p_times(2, 1);
    } else {
        p_times(1, 0);
        p_times(0, 0);
        p_times(1, 1);
        p_times(2, 2);
    }
    __syncthreads();
    if (warp == 0) p_times(3, 0);
    else if (warp == 1) p_times(2, 0);
    else if (warp == 2) p_times(3, 2);
    else p_times(3, 3);
}

// The walk.  Eight warps own 16 value columns of a head: four carry the state
// (each a quarter of its rows, in registers), four make the outputs; a block
// has NG such groups, which share the chunk's tiles, and four warps that load the
// next two chunks' while this one's are in use.  All products are taken
// transposed, with the 16 columns as the MMA's m:
//   R^T = V^T - (S0^T K^T) diag(ck);  U^T = R^T T^T;  S'^T = keep S0^T + (U^T diag(cs)) K
// by the state's warps, each for 16 tokens or a quarter of the rows, with R, U
// and S changing hands through shared memory, and beside them
//   O^T = (S0^T Q^T) diag(cq) + R^T (P T)^T.
// A product of S waits for the chunk before it, so a walk's speed is this chain of
// three small products, not its operations; taking the outputs out of it and
// keeping 16 columns a group makes it as short as the MMA allows.  Warp w and
// the output warp beside it on the same scheduler take tokens 16 w and 16 (3 - w), so
// that the triangles' work adds up to the same on each.
//
// 8000 tokens of 16 heads, one group a block: 170 us, 1.35 us a chunk (the operator's bytes would take 20), with
// shared memory busy in three quarters of the cycles, most of that for fragments of S that eight warps
// need; two groups 2.3 us a chunk (24 bytes of a thread's registers spilled).
template <int DK, int NG>
struct Scan {
    static constexpr int kThreads = NG * 256 + 128;
    static constexpr int kTile = kChunk * DK * 2;
    static constexpr int kRecord = 2 * kTile;
    static constexpr int kLoPart = 2 * kTri * 2;                 // from the record's hi to its lo
    static constexpr int kScales = kRecord + 2 * kLoPart;
    static constexpr int kV = kRecord + sizeof(Chunk);
    static constexpr int kStage = kV + kChunk * NG * 32;
    static constexpr int kSx = 16 * DK * 2;
    static constexpr int kRx = 16 * kChunk * 2;
    static constexpr int kGroup = 2 * kSx + 4 * kRx;
    static constexpr int kStages = 3;
    static constexpr int kSmem = kStages * kStage + NG * kGroup;
};

template <int DK, int NG>
__global__ void __launch_bounds__(NG * 256 + 128, 1) scan_kernel(const DeltaArgs a, const Chunk* chunks) {
    using C = Scan<DK, NG>;
    constexpr int kVecs = DK / 8;
    constexpr int kN = DK / 32;       // n8 tiles of a state warp's rows
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t landed[C::kStages];
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::kStages; ++i) mbar_init(&landed[i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31;
    const int g = lane >> 2, t = lane & 3;
    const int h = blockIdx.y, b = blockIdx.z;
    const int col0 = blockIdx.x * NG * 16;
    int begin, end, slot;
    if (!sequence(a, b, begin, end, slot)) return;
    const int chunks_here = (end - begin + kChunk - 1) / kChunk;
    const uint32_t base = smem_u32(smem);

    if (tid >= NG * 256) {
        // ---- the loading warps: two chunks ahead ----
        constexpr int kStep = 128 / kVecs;           // rows of one sweep of the 128 threads; a multiple of 8,
        static_assert(kStep % 8 == 0, "swizzle");    // so a thread keeps its place in the swizzle
        const int kh = h / a.share, lt = tid - NG * 256;
        const int lr = lt / kVecs, lx = lt % kVecs;
        const __half* kp = a.k + static_cast<int64_t>(begin + lr) * a.k_ts + kh * a.k_hs + lx * 8;
        const __half* qp = a.q + static_cast<int64_t>(begin + lr) * a.q_ts + kh * a.q_hs + lx * 8;
        const int64_t k_step = kStep * a.k_ts, q_step = kStep * a.q_ts;
        const Chunk* rec = chunks + first_chunk(begin, b) * a.v_heads + h;
        bool dead = false;
        auto issue = [&](int c) {
            if (c < chunks_here) {
                const int st = c % C::kStages;
                const uint32_t stage = base + st * C::kStage;
                if (lt == 0) {
                    fence_proxy_async_smem();      // the stage's reads come before the copy into it
                    mbar_expect_tx(&landed[st], kChunkBytes);
                    bulk_load(smem + st * C::kStage + C::kRecord, rec, kChunkBytes, &landed[st]);
                }
                rec += a.v_heads;
                const uint32_t dst = tile_at<kVecs>(stage, lr, lx);
                const int t0 = begin + c * kChunk;
                const int n = min(kChunk, end - t0);
#pragma unroll
                for (int i = 0; i < kChunk / kStep; ++i) {
                    const bool ok = i * kStep + lr < n;
                    cp_async16_or_zero(dst + i * kStep * kVecs * 16, ok ? kp : a.k, ok);
                    cp_async16_or_zero(dst + i * kStep * kVecs * 16 + C::kTile, ok ? qp : a.q, ok);
                    kp += k_step;
                    qp += q_step;
                }
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const int item = i * 128 + lt, r = item / (2 * NG), x = item % (2 * NG);
                    const bool ok = r < n && col0 + x * 8 < a.dv;
                    cp_async16_or_zero(tile_at<2 * NG>(stage + C::kV, r, x),
                                       ok ? a.v + static_cast<int64_t>(t0 + r) * a.v_ts + h * a.v_hs + col0 + x * 8 : a.v, ok);
                }
            }
            cp_async_commit();
        };
        issue(0);
        issue(1);
#pragma unroll 1
        for (int c = 0; c < chunks_here; ++c) {
            cp_async_wait<1>();
            if (lt == 0 && !dead && !mbar_wait(&landed[c % C::kStages], (c / C::kStages) & 1)) {
                dead = true;      // gives up waiting, not the barriers: the block still ends
                atomicOr(&g_gated_delta_dev_error, kDevErrTimeout);
            }
            __syncthreads();   // chunk c is there, and c - 1 is done with
            issue(c + 2);
        }
        return;
    }

    const int group = tid >> 8, warp = (tid >> 5) & 3;
    const bool outputs = (tid >> 7) & 1;
    const int col = col0 + group * 16;
    const bool live = col < a.dv;
    const uint32_t s_hi = base + C::kStages * C::kStage + group * C::kGroup, s_lo = s_hi + C::kSx, r_hi = s_lo + C::kSx,
                   r_lo = r_hi + C::kRx, w_hi = r_lo + C::kRx, w_lo = w_hi + C::kRx;
    const int blk = outputs ? 3 - warp : warp;       // this warp's 16 tokens of a chunk
    const int a_row = lane & 15, a_vec = lane >> 4;                                // A operand
    const int b_row = (lane & 7) + (lane >> 4) * 8, b_vec = (lane >> 3) & 1;       // B operand, rows = n
    const uint32_t tri_row = blk * 512 + lane * 16;       // this lane's row of block (blk, j) of a triangle, from block (0, j)
    auto state_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + 2 * group) : "memory"); };
    auto group_sync = [&]() { asm volatile("bar.sync %0, 256;" ::"r"(2 + 2 * group) : "memory"); };
    auto scale_pair = [&](uint32_t sc, int which, int n) {
        float2 x;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                     : "=f"(x.x), "=f"(x.y)
                     : "r"(sc + (which * kChunk + blk * 16 + n * 8 + 2 * t) * 4));
        return x;
    };
    auto put = [&](uint32_t at, uint32_t x) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(x) : "memory"); };

    if (outputs) {
        for (int c = 0; c < chunks_here; ++c) {
            __syncthreads();
            const uint32_t stage = base + c % C::kStages * C::kStage, sc = stage + C::kScales;
            const uint32_t p_hi = stage + C::kRecord + kTri * 2 + tri_row;
            float o[2][4], ol[2][4], x[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][e] = ol[n][e] = x[n][e] = 0.0f;
#pragma unroll
            for (int kk = 0; kk < DK / 16; ++kk) {
                uint32_t sh[4], sl[4], qf[4];
                ldsm4(sh, tile_at<kVecs>(s_hi, a_row, kk * 2 + a_vec));
                ldsm4(sl, tile_at<kVecs>(s_lo, a_row, kk * 2 + a_vec));
                ldsm4(qf, tile_at<kVecs>(stage + C::kTile, blk * 16 + b_row, kk * 2 + b_vec));
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    mma16816(o[n], sh, qf[2 * n], qf[2 * n + 1]);
                    mma16816(ol[n], sl, qf[2 * n], qf[2 * n + 1]);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const float2 cq = scale_pair(sc, 1, n);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[n][e] = (e & 1 ? cq.y : cq.x) * (o[n][e] + kLoInv * ol[n][e]);
                    ol[n][e] = 0.0f;
                }
            }
            group_sync();       // R is there, and S0 has been read
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j > blk) break;
                uint32_t rh[4], rl[4], ph[4], pl[4];
                ldsm4(rh, tile_at<8>(r_hi, a_row, j * 2 + a_vec));
                ldsm4(rl, tile_at<8>(r_lo, a_row, j * 2 + a_vec));
                ldsm4(ph, p_hi + tri_block(0, j) * 512);
                ldsm4(pl, p_hi + C::kLoPart + tri_block(0, j) * 512);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    mma16816(x[n], rh, ph[2 * n], ph[2 * n + 1]);
                    mma16816(ol[n], rl, ph[2 * n], ph[2 * n + 1]);
                    mma16816(ol[n], rh, pl[2 * n], pl[2 * n + 1]);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int tok = begin + c * kChunk + blk * 16 + n * 8 + g;
                const float2 oq = scale_pair(sc, 3, n);
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    // 8x8 transpose: lane (g, t) then has token g, columns 2t, 2t + 1
                    const uint32_t r = movm_t(h2_as_u32(__floats2half2_rn(o[n][e] + oq.x * (x[n][e] + kLoInv * ol[n][e]),
                                                                           o[n][e + 1] + oq.y * (x[n][e + 1] + kLoInv * ol[n][e + 1]))));
                    if (live && tok < end)
                        *reinterpret_cast<uint32_t*>(a.out + (static_cast<int64_t>(tok) * a.v_heads + h) * a.dv + col +
                                                     e * 4 + 2 * t) = r;
                }
            }
        }
        return;
    }

    // ---- the state's warps ----
    // S^T as C fragments: rows (columns of the state) g, g + 8, columns (its rows)
    // warp * DK / 4 + 8 n + 2t, + 1
    float s[kN][4];
    const int64_t at = ((static_cast<int64_t>(slot) * a.v_heads + h) * DK + warp * (DK / 4) + 2 * t) * a.dv + col + g;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            s[n][e] = a.state_in && live ? a.state_in[at + static_cast<int64_t>(n * 8 + (e & 1)) * a.dv + (e >> 1) * 8] : 0.0f;
    auto put_state = [&]() {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                uint32_t hi, lo;
                split_scaled(s[n][e], s[n][e + 1], hi, lo);
                put(tile_at<kVecs>(s_hi, g + e * 4, warp * kN + n) + t * 4, hi);
                put(tile_at<kVecs>(s_lo, g + e * 4, warp * kN + n) + t * 4, lo);
            }
    };
    auto put_rows = [&](uint32_t hi_at, uint32_t lo_at, const float (&x)[2][4]) {
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                uint32_t hi, lo;
                split_scaled(x[n][e], x[n][e + 1], hi, lo);
                put(tile_at<8>(hi_at, g + e * 4, warp * 2 + n) + t * 4, hi);
                put(tile_at<8>(lo_at, g + e * 4, warp * 2 + n) + t * 4, lo);
            }
    };
    put_state();
    for (int c = 0; c < chunks_here; ++c) {
        __syncthreads();
        const uint32_t stage = base + c % C::kStages * C::kStage, sc = stage + C::kScales;
        const uint32_t t_hi = stage + C::kRecord + tri_row;

        // S0^T K^T for this warp's tokens
        float x[2][4], xl[2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[n][e] = xl[n][e] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < DK / 16; ++kk) {
            uint32_t sh[4], sl[4], kf[4];
            ldsm4(sh, tile_at<kVecs>(s_hi, a_row, kk * 2 + a_vec));
            ldsm4(sl, tile_at<kVecs>(s_lo, a_row, kk * 2 + a_vec));
            ldsm4(kf, tile_at<kVecs>(stage, blk * 16 + b_row, kk * 2 + b_vec));
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                mma16816(x[n], sh, kf[2 * n], kf[2 * n + 1]);
                mma16816(xl[n], sl, kf[2 * n], kf[2 * n + 1]);
            }
        }
        uint32_t vf[4];
        ldsm4_t(vf, tile_at<2 * NG>(stage + C::kV, blk * 16 + b_row, group * 2 + b_vec));
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const float2 ck = scale_pair(sc, 0, n);
            const float2 v0 = __half22float2(u32_as_h2(vf[2 * n])), v1 = __half22float2(u32_as_h2(vf[2 * n + 1]));
            x[n][0] = v0.x - ck.x * (x[n][0] + kLoInv * xl[n][0]);
            x[n][1] = v0.y - ck.y * (x[n][1] + kLoInv * xl[n][1]);
            x[n][2] = v1.x - ck.x * (x[n][2] + kLoInv * xl[n][2]);
            x[n][3] = v1.y - ck.y * (x[n][3] + kLoInv * xl[n][3]);
        }
        put_rows(r_hi, r_lo, x);
        group_sync();

        // U^T = R^T T^T
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[n][e] = xl[n][e] = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > blk) break;
            uint32_t rh[4], rl[4], th[4], tl[4];
            ldsm4(rh, tile_at<8>(r_hi, a_row, j * 2 + a_vec));
            ldsm4(rl, tile_at<8>(r_lo, a_row, j * 2 + a_vec));
            ldsm4(th, t_hi + tri_block(0, j) * 512);
            ldsm4(tl, t_hi + C::kLoPart + tri_block(0, j) * 512);
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                mma16816(x[n], rh, th[2 * n], th[2 * n + 1]);
                mma16816(xl[n], rl, th[2 * n], th[2 * n + 1]);
                mma16816(xl[n], rh, tl[2 * n], tl[2 * n + 1]);
            }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const float2 cs = scale_pair(sc, 2, n);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[n][e] = (e & 1 ? cs.y : cs.x) * (x[n][e] + kLoInv * xl[n][e]);
        }
        put_rows(w_hi, w_lo, x);
        state_sync();

        // S'^T = keep S0^T + (U^T diag(cs)) K
        float keep, sl[kN][4];
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(keep) : "r"(sc + 4 * kChunk * 4));
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[n][e] *= keep;
                sl[n][e] = 0.0f;
            }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t wh[4], wl[4];
            ldsm4(wh, tile_at<8>(w_hi, a_row, j * 2 + a_vec));
            ldsm4(wl, tile_at<8>(w_lo, a_row, j * 2 + a_vec));
#pragma unroll
            for (int p = 0; p < kN / 2; ++p) {
                uint32_t kf[4];
                ldsm4_t(kf, tile_at<kVecs>(stage, j * 16 + a_row, warp * kN + p * 2 + a_vec));
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    mma16816(s[2 * p + n], wh, kf[2 * n], kf[2 * n + 1]);
                    mma16816(sl[2 * p + n], wl, kf[2 * n], kf[2 * n + 1]);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] += kLoInv * sl[n][e];
        put_state();
    }
    // a value beyond fp16's range makes an operand infinite and its low part too, and so the state NaN for good
    bool finite = true;
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) finite &= isfinite(s[n][e]);
    if (!finite && chunks_here > 0) atomicOr(&g_gated_delta_dev_error, kDevErrRange);
    if (a.state_out && live) {
#pragma unroll
        for (int n = 0; n < kN; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                a.state_out[at + static_cast<int64_t>(n * 8 + (e & 1)) * a.dv + (e >> 1) * 8] = s[n][e];
    }
}

// ---- the same walk on the tcgen05 tensor cores, for many heads -----------------------
//
// One block per head (128 value columns), the columns as the MMA's M = 128 rows:
//   D1 = S^T [K; Q]^T;  D2 = R^T [T; P T]^T;  D3 = W^T K  with W = diag(cs) U,
// the left operands from tensor memory (a shared-memory operand each side would take
// all of its bandwidth): S beside the accumulators, R and W as hi and lo in the place
// of the halves of D1 and D2 that they are made from.  K's tile of tokens by rows serves
// both as [K; Q] and, read with N contiguous, as W's factor; a block column of a
// triangle is an operand of the rows from its diagonal on.  The state itself lives
// in D3: keep S is put there before the product adds to it.
//
// A row of an accumulator, one value column, belongs to one thread of each of
// four warpgroups (a quarter of the tokens and of the state's rows each), which turn
// D1 into R, D2 into W and D3 into the next S; four warps write the outputs from the
// other halves of D1 and D2, whose products follow the state's, three load up to
// three chunks ahead, one issues the MMAs, 16 of K at a time as soon as that part
// of an operand is there.  The passes over the accumulators are what a chunk waits for,
// so they are short rolled loops (straight code is fetched more slowly than it
// runs) on many warps.
//
// A chunk takes 3.1 us (5800 clocks at DK = 128: E1 and E2, to R and to W, 1250 and 550, the
// products before them 700 and 600, the state's product 950, its pass 1500): 15100 warp
// instructions, 66 % of the issue slots, tensor pipe 35 %.  7600 clocks with both
// halves of a product in one, two stages, and copies that a warp waited for.
//
// A split operand is hi + 2^-11 lo here too, in one accumulator: the products with a
// lo come first, and the first one with a hi scales what is there by 2^-11 (the MMA's
// scaling of its input).  A row's values are first multiplied by a power of two that
// keeps a bound of all of a chunk's,
// |S|, |S'|, |R|, |U| <= sqrt(Dk) max|S| + (C + 1) max|v|, between 2^9 and 2^13 (the
// state's update is a contraction).  max|S| is measured every fourth chunk and
// raised by C max|v| for each chunk since, so that the scale is there before the
// state is; the state stays in its scale in registers.  So values keep 22 bits, or an
// absolute 2^-45 of the bound (2^-36 in this scale) where that is more, and a factor
// of 8 above the bound stays below fp16's end.  (With lo in the scale of hi the absolute
// error is 2^-29 of the bound: too much for small values beside one of 30000.  The low parts'
// scaling costs 3 % of a chunk's time, all of it in the passes.)
template <int DK>
struct Walk {
    static constexpr int kLoaders = 96;           // three warps
    static constexpr int kThreads = 768;          // state 16 warps, outputs 4, loading 3, MMA issue 1
    static constexpr int kSub = DK / 64;          // 128-byte tiles of 64 dims
    static constexpr int kTile = 128 * 128;
    static constexpr int kTp = kSub * kTile;      // [K; Q], then the chunk's record: triangles and scales
    static constexpr int kScales = kTp + kTriBytes;
    static constexpr int kV = kTp + 22 * 1024;    // 64 tokens of 128 values
    static constexpr int kStage = kV + kChunk * 256;
    static constexpr int kStages = 3;
    static constexpr int kSmem = kStages * kStage + 1024;
    static constexpr int kPart = DK / 4;          // state rows of a thread
    static constexpr int kBatches = kPart / 16;
    // tensor-memory columns
    static constexpr uint32_t kD1 = 0, kD2 = 128, kD3 = 256, kSHi = 384, kSLo = 448;
    static_assert(kChunkBytes <= 22 * 1024 && kStage % 1024 == 0 && kSmem <= 232448 - 16384, "shared memory");
};

__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// As mbar_wait, suspended for up to 1 ms at a time: a hint, the hardware may come back sooner, so the clock bounds the wait.
__device__ __forceinline__ bool mbar_wait_suspended(uint64_t* bar, uint32_t parity) {
    uint64_t t0 = 0;
#pragma unroll 1
    for (uint32_t i = 0;; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
            : "memory");
        if (ok) return true;
        if (i & 7) continue;
        const uint64_t now = globaltimer_ns();
        if (i == 0) t0 = now;
        else if (now - t0 > 2000000000ull) return false;
    }
}
// 16 columns of this warp's 32 lanes, to be waited for with tmem_wait.
__device__ __forceinline__ void tmem_get(uint32_t addr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
// Waits for all tmem_get so far; `r` are the ones used next.
template <int N>
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
// Arrives when all of this thread's cp.async so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// The power of two that takes a bound of a row's values to 2^11 .. 2^12, and its inverse.
__device__ __forceinline__ float2 row_scale(float bound) {
    const int e = min(max(138 - static_cast<int>((__float_as_uint(bound) >> 23) & 255u), -100), 100);
    return make_float2(__uint_as_float(static_cast<uint32_t>(127 + e) << 23), __uint_as_float(static_cast<uint32_t>(127 - e) << 23));
}

// K-major operand of 8x8 matrices of 128 bytes without swizzle: the next 8 of K 128
// bytes on, the next 8 rows 256.
__device__ __forceinline__ uint64_t smem_desc_plain(uint32_t saddr) {
    return static_cast<uint64_t>((saddr >> 4) & 0x3fffu) | (static_cast<uint64_t>(128 >> 4) << 16) |
           (static_cast<uint64_t>(256 >> 4) << 32) | (static_cast<uint64_t>(1u) << 46);
}

template <int DK>
__global__ void __launch_bounds__(Walk<DK>::kThreads, 1) walk_kernel(const DeltaArgs a, const Chunk* chunks) {
    using C = Walk<DK>;
    constexpr int kVecs = DK / 8;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[C::kStages], empty[C::kStages], s_ready[2], r_ready, w_ready, made[4], o_done, scaled;
    __shared__ float2 most[3][4][128];      // [chunk % 3][part][row]: max|S|, max|v|
    __shared__ __align__(16) float out_scales[2][2 * kChunk];      // [chunk % 2]: cq, oq
    __shared__ uint32_t tmem_slot;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* smem = smem_raw + (base - smem_u32(smem_raw));
    if (warp == 23) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) {
            mbar_init(&full[i], C::kLoaders + 1);      // the loading threads, and the announcement of the bulk copy
            mbar_init(&empty[i], 21);      // state and output warps, and the MMAs
        }
        for (int i = 0; i < 2; ++i) mbar_init(&s_ready[i], 16);
        mbar_init(&r_ready, 16);
        mbar_init(&w_ready, 16);
        for (int i = 0; i < 4; ++i) mbar_init(&made[i], 1);
        mbar_init(&o_done, 4);
        mbar_init(&scaled, 16);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_trigger();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    pdl_wait();

    const int h = blockIdx.y, col0 = blockIdx.x * 128;
    int b = blockIdx.z;
    if (a.batch > 1 && a.batch <= 32) {
        // The longest sequences first: a long one begun when the others end is waited for alone (12 sequences of 50 to
        // 4000 tokens of 16 heads: 317 us, in their own order 378).  Each warp ranks them by itself; more than a
        // warp's lanes even out (100 sequences up to 500 tokens, ranked by the block, took 2 % longer).
        const int mine = lane < a.batch ? a.cu[lane + 1] - a.cu[lane] : 0;
        int rank = 0;
        for (int i = 0; i < a.batch; ++i) {
            const int other = __shfl_sync(0xffffffffu, mine, i);
            rank += other > mine || (other == mine && i < lane);
        }
        b = __ffs(__ballot_sync(0xffffffffu, lane < a.batch && rank == b)) - 1;
    }
    int begin = 0, end = 0, slot = 0;
    const bool valid = sequence(a, b, begin, end, slot);
    const int chunks_here = valid ? (end - begin + kChunk - 1) / kChunk : 0;
    // Every wait is bounded.  A thread whose wait gave up records it and goes on
    // without waiting, so that all barriers still meet and the block ends.  Warps
    // wait whole and suspended: one lane of each of 23 asking again and again took
    // a fifth of a chunk's time from the thread that issues, which alone does ask.
    bool dead = false;
    auto gave_up = [&]() {
        dead = true;
        atomicOr(&g_gated_delta_dev_error, kDevErrTimeout);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!dead && !mbar_wait_suspended(bar, parity & 1)) gave_up();
    };
    auto wait_one = [&](uint64_t* bar, uint32_t parity) {
        if (!dead && !mbar_wait(bar, parity & 1)) gave_up();
    };
    auto scales_of = [&](int c) { return reinterpret_cast<const float*>(smem + c % C::kStages * C::kStage + C::kScales); };
    // A row's scale and its inverse, chunk by chunk.
    struct Scale {
        float s = 0.0f, v = 0.0f;      // bound of the state before the chunk; max|v| of the chunk
        float2 now = make_float2(0.0f, 0.0f);
        __device__ __forceinline__ float2 next(int c, const float2 (&most)[4][128], int row) {
            float2 m = most[0][row];
#pragma unroll
            for (int p = 1; p < 4; ++p) m = make_float2(fmaxf(m.x, most[p][row].x), fmaxf(m.y, most[p][row].y));
            // measured at the start and behind chunks 0, 4, 8, ..., known one chunk later
            if (c == 0 || (c >= 2 && (c & 3) == 2)) s = (DK == 128 ? 11.4f : 8.1f) * m.x;
            s += kChunk * v;
            v = m.y;
            const float bound = s + (kChunk + 1) * v, at = bound * now.x;
            if (!(at >= 512.0f && at < 8192.0f)) now = row_scale(bound);
            return now;
        }
    };

    if (warp < 16) {
        // ---- the state ----
        const int part = warp >> 2, row = (warp & 3) * 32 + lane;
        const int col = col0 + row;
        const bool live = col < a.dv && valid;
        const uint32_t lane_at = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const int64_t at = ((static_cast<int64_t>(slot) * a.v_heads + h) * DK + part * C::kPart) * a.dv + col;
        const unsigned char* v_at = smem + C::kV + part * 16 * 256 + row * 2;      // this thread's 16 tokens
        float most_s = 0.0f;
        // 16 state rows of this part (batch b) as hi and lo operand, and times `kept` = 2^11 keep where the product, its
        // low part first, adds to them
        auto put_state = [&](int b, const float (&x)[16], float kept) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) split_scaled(x[2 * i], x[2 * i + 1], hi[i], lo[i]);
            tmem_st8(lane_at + C::kSHi + part * (C::kPart / 2) + b * 8, hi);
            tmem_st8(lane_at + C::kSLo + part * (C::kPart / 2) + b * 8, lo);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    float a = x[e * 8 + i], b = x[e * 8 + i + 1];
                    mul2(a, b, kept, kept);
                    hi[i] = __float_as_uint(a), hi[i + 1] = __float_as_uint(b);
                }
                tmem_st8(lane_at + C::kD3 + part * C::kPart + b * 16 + e * 8, hi);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_ready[b]);
        };
        // R or W of this part's 16 tokens as hi and lo operand, in the place of the product that it was made from
        auto put_row = [&](const float (&x)[16], uint32_t place, uint64_t* ready) {
            uint32_t hi[8], lo[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) split_scaled(x[2 * i], x[2 * i + 1], hi[i], lo[i]);
            tmem_st8(lane_at + place + part * 16, hi);
            tmem_st8(lane_at + place + part * 16 + 8, lo);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ready);
        };
        // This thread's part of a chunk's max|v| and its own max|S|, for the row's other threads and the outputs
        auto measure_row = [&](int c) {
            wait(&full[c % C::kStages], c / C::kStages);
            const unsigned char* p = v_at + c % C::kStages * C::kStage;
            __half m = __float2half_rn(0.0f);
#pragma unroll
            for (int i = 0; i < 16; ++i) m = __hmax(m, __habs(*reinterpret_cast<const __half*>(p + i * 256)));
            most[c % 3][part][row] = make_float2(most_s, __half2float(m));
        };
        Scale scale;
        auto agree = [&](int c) {
            asm volatile("bar.sync 1, 512;" ::: "memory");
            if (lane == 0) mbar_arrive(&scaled);
            return scale.next(c, most[c % 3], row);
        };
        float2 now = make_float2(1.0f, 1.0f);      // registers and operands of chunk c are in its scale
        if (chunks_here == 0 && a.state_out && live) {
            for (int i = 0; i < C::kPart; ++i)
                a.state_out[at + static_cast<int64_t>(i) * a.dv] = a.state_in ? a.state_in[at + static_cast<int64_t>(i) * a.dv] : 0.0f;
        }
        if (chunks_here > 0) {
            float x[C::kBatches][16];
#pragma unroll
            for (int i = 0; i < C::kPart; ++i) {
                x[i / 16][i % 16] = a.state_in && live ? a.state_in[at + static_cast<int64_t>(i) * a.dv] : 0.0f;
                most_s = fmaxf(most_s, fabsf(x[i / 16][i % 16]));
            }
            measure_row(0);
            now = agree(0);
            const float kept = kLo * scales_of(0)[4 * kChunk];
#pragma unroll
            for (int b = 0; b < C::kBatches; ++b) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[b][i] *= now.x;
                put_state(b, x[b], kept);
            }
        }

#pragma unroll 1
        for (int c = 0; c < chunks_here; ++c) {
            const float* sc = scales_of(c) + part * 16;
            float x[16];
            wait(&made[0], c);
            tc_fence_after();
            tmem_ld16(lane_at + C::kD1 + part * 16, x);
            const unsigned char* vp = v_at + c % C::kStages * C::kStage;
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 ck = *reinterpret_cast<const float4*>(sc + i);
                const float* cp = &ck.x;
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    float v0 = __half2float(*reinterpret_cast<const __half*>(vp + (i + e) * 256));
                    float v1 = __half2float(*reinterpret_cast<const __half*>(vp + (i + e + 1) * 256));
                    mul2(v0, v1, now.x, now.x);
                    x[i + e] = v0 - cp[e] * x[i + e];
                    x[i + e + 1] = v1 - cp[e + 1] * x[i + e + 1];
                }
            }
            put_row(x, C::kD1, &r_ready);
            const bool last = c + 1 == chunks_here;
            if (!last) measure_row(c + 1);      // while U is made
            wait(&made[1], c);
            tc_fence_after();
            tmem_ld16(lane_at + C::kD2 + part * 16, x);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 cs = *reinterpret_cast<const float4*>(sc + 2 * kChunk + i);
                mul2(x[i], x[i + 1], cs.x, cs.y);
                mul2(x[i + 2], x[i + 3], cs.z, cs.w);
            }
            put_row(x, C::kD2, &w_ready);
            if (lane == 0) mbar_arrive(&empty[c % C::kStages]);
            // while the last product is made: the next chunk's scale and decay
            float2 next = now;
            float kept = 0.0f;
            if (!last) {
                next = agree(c + 1);
                kept = kLo * scales_of(c + 1)[4 * kChunk];
            }
            const float change = next.x * now.y;
            const bool changes = __any_sync(0xffffffffu, change != 1.0f), measure = (c & 3) == 0;
            if (measure) most_s = 0.0f;
            wait(&made[2], c);
            tc_fence_after();
#pragma unroll 1
            for (int b = 0; b < C::kBatches; ++b) {
                tmem_ld16(lane_at + C::kD3 + part * C::kPart + b * 16, x);
                if (measure) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) most_s = fmaxf(most_s, fabsf(x[i]));
                }
                if (last) {
                    bool finite = true;
#pragma unroll
                    for (int i = 0; i < 16; ++i) finite &= isfinite(x[i]);
                    if (!finite) atomicOr(&g_gated_delta_dev_error, kDevErrRange);
                    if (a.state_out && live) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) a.state_out[at + static_cast<int64_t>(b * 16 + i) * a.dv] = x[i] * now.y;
                    }
                    continue;
                }
                if (changes) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] *= change;
                }
                put_state(b, x, kept);
            }
            if (measure) most_s *= now.y;
            now = next;
        }
    } else if (warp < 20) {
        // ---- the outputs ----
        const int row = (warp & 3) * 32 + lane;
        const int col = col0 + row;
        const uint32_t lane_at = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        Scale scale;
        // "done" also says that the next chunk's scale has been seen, so the state cannot get ahead by two
        if (chunks_here > 0) wait(&scaled, 0);
        if (lane == 0) mbar_arrive(&o_done);
        const int odd = lane & 1;
        // two lanes swap values: the even one writes both columns of the first of two tokens, the odd one of the second
        const int64_t step = 2 * static_cast<int64_t>(a.v_heads) * a.dv;
        __half* to = a.out + ((static_cast<int64_t>(begin) + odd) * a.v_heads + h) * a.dv + (col & ~1);
        for (int c = 0; c < chunks_here; ++c) {
            // the outputs are done last: their scales are copied, and the stage is free for the next chunk before that
            float* sc = out_scales[c & 1];
            wait(&full[c % C::kStages], c / C::kStages);
            sc[row] = scales_of(c)[(row < kChunk ? kChunk : 2 * kChunk) + row];
            asm volatile("bar.sync 2, 128;" ::: "memory");
            if (lane == 0) mbar_arrive(&empty[c % C::kStages]);
            const float unit = scale.next(c, most[c % 3], row).y;
            wait(&made[3], c);
            tc_fence_after();
            const int left = col < a.dv ? end - begin - c * kChunk - odd : 0;      // of this lane's tokens
#pragma unroll 1
            for (int b = 0; b < 4; ++b) {
                uint32_t x[16], y[16];
                tmem_get(lane_at + C::kD1 + 64 + b * 16, x);
                tmem_get(lane_at + C::kD2 + 64 + b * 16, y);
                float cq[16], oq[16], o[16];
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    *reinterpret_cast<float4*>(cq + i) = *reinterpret_cast<const float4*>(sc + b * 16 + i);
                    *reinterpret_cast<float4*>(oq + i) = *reinterpret_cast<const float4*>(sc + kChunk + b * 16 + i);
                }
                tmem_wait(x);
                tmem_wait(y);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = unit * (cq[i] * __uint_as_float(x[i]) + oq[i] * __uint_as_float(y[i]));
                __half2 r[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float other = __shfl_xor_sync(0xffffffffu, odd ? o[2 * i] : o[2 * i + 1], 1);
                    r[i] = odd ? __floats2half2_rn(other, o[2 * i + 1]) : __floats2half2_rn(o[2 * i], other);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (b * 16 + 2 * i < left) *reinterpret_cast<__half2*>(to + i * step) = r[i];
                to += 8 * step;
            }
            if (c + 1 < chunks_here) wait(&scaled, c + 1);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_done);
        }
    } else if (warp < 23) {
        // ---- loading ----
        const int kh = h / a.share, lt = tid - 20 * 32;
        const __half* k0 = a.k + kh * a.k_hs;
        const __half* q0 = a.q + kh * a.q_hs;
        const __half* v0 = a.v + h * a.v_hs + col0;
        const Chunk* rec = chunks + first_chunk(begin, b) * a.v_heads + h;
        // rows of `vecs` vectors of 16 bytes, `n` of them there, one vector of every few rows per thread
        auto copy_rows = [&](uint32_t to, const __half* from, int64_t stride, auto vecs, int n, bool live, auto place) {
            constexpr int kStep = C::kLoaders / decltype(vecs)::value;
            const int x = lt % decltype(vecs)::value;
            const __half* p = from + (lt / decltype(vecs)::value) * stride + x * 8;
#pragma unroll 2
            for (int r = lt / decltype(vecs)::value; r < kChunk; r += kStep, p += kStep * stride) {
                const bool ok = live && r < n;
                cp_async16_or_zero(to + place(r, x), ok ? p : from, ok);
            }
        };
        auto swizzled = [](int r, int x) { return static_cast<uint32_t>((x >> 3) * C::kTile + r * 128 + (((x & 7) ^ (r & 7)) << 4)); };
        auto plain = [](int r, int x) { return static_cast<uint32_t>(r * 256 + x * 16); };
        using Vecs = std::integral_constant<int, kVecs>;
        using VVecs = std::integral_constant<int, 16>;
        const bool v_live = col0 + (lt & 15) * 8 < a.dv;
        for (int c = 0; c < chunks_here; ++c) {
            const int st = c % C::kStages;
            if (c >= C::kStages) wait(&empty[st], c / C::kStages - 1);
            const uint32_t stage = base + st * C::kStage;
            fence_proxy_async_smem();      // the stage's reads come before the copies into it
            if (lt == 0) {
                mbar_expect_tx(&full[st], kChunkBytes);
                bulk_load(smem + st * C::kStage + C::kTp, rec, kChunkBytes, &full[st]);
            }
            rec += a.v_heads;
            const int64_t t0 = begin + c * kChunk;
            const int n = min(kChunk, end - begin - c * kChunk);
            copy_rows(stage, k0 + t0 * a.k_ts, a.k_ts, Vecs(), n, true, swizzled);
            copy_rows(stage + kChunk * 128, q0 + t0 * a.q_ts, a.q_ts, Vecs(), n, true, swizzled);
            copy_rows(stage + C::kV, v0 + t0 * a.v_ts, a.v_ts, VVecs(), n, v_live, plain);
            cp_async_arrive(&full[st]);      // once this thread's copies have landed
        }
        // all copies have landed before the block's shared memory goes
        for (int c = max(0, chunks_here - C::kStages); c < chunks_here; ++c) wait(&full[c % C::kStages], c / C::kStages);
    } else {
        // ---- MMA issue ----
        // The warp stays together and an elected lane issues: 36 clocks an MMA beside 23 busy warps (74 from a
        // branch of lane 0, 130 from a rolled loop).
        constexpr uint32_t kIdesc = instr_desc_f16(128, kChunk), kIdescT = instr_desc_f16(128, DK) | (1u << 16);   // B with N contiguous
        constexpr uint64_t kQ = (kChunk * 128) >> 4;      // from K to Q
        // descriptors count in 16 bytes; all are constants away from these
        const uint64_t tiles = smem_desc_sw128(base);
        const uint64_t tri = smem_desc_plain(base + C::kTp);
        // K by tokens: groups of eight 1024 bytes apart, the second 64 dims a tile on
        const uint64_t turned = (tiles & ~(static_cast<uint64_t>(0x3fff) << 16)) | (static_cast<uint64_t>(C::kTile >> 4) << 16);
        for (int c = 0; c < chunks_here; ++c) {
            const uint64_t st = static_cast<uint64_t>(c % C::kStages * (C::kStage >> 4));
            const uint64_t kq = tiles + st, tp = tri + st, kt = turned + st;
            // products with a low part first, each accumulator brought to scale by its first product with a high part
            auto state_low = [&](int k, int half) {
                const uint64_t d = kq + half * kQ + (((k >> 2) * C::kTile + (k & 3) * 32) >> 4);
                mma_f16_ts(tmem + C::kD1 + half * kChunk, tmem + C::kSLo + k * 8, d, kIdesc, k > 0);
            };
            auto state_high = [&](int half) {
#pragma unroll
                for (int k = 0; k < DK / 16; ++k) {
                    const uint64_t d = kq + half * kQ + (((k >> 2) * C::kTile + (k & 3) * 32) >> 4);
                    const uint32_t to = tmem + C::kD1 + half * kChunk;
                    if (k == 0) mma_f16_ts_shifted<kLoBits>(to, tmem + C::kSHi, d, kIdesc);
                    else mma_f16_ts(to, tmem + C::kSHi + k * 8, d, kIdesc, 1);
                }
            };
            // 16 tokens reach the outputs from themselves on; the first 16 reach all, so their products begin and scale
            auto row_product = [&](int half) {
#pragma unroll
                for (int step = 0; step < 8; ++step) {
                    const int k = step & 3;
                    const uint32_t to = tmem + C::kD2 + half * kChunk + k * 16, r = tmem + C::kD1 + k * 16;
                    const uint32_t idesc = instr_desc_f16(128, kChunk - k * 16);
                    const uint64_t hi = tp + ((half * kTri * 2 + tri_column(k) * 512) >> 4), lo = hi + ((2 * kTri * 2) >> 4);
                    if (step < 4) {
                        mma_f16_ts(to, r + 8, hi, idesc, k > 0);
                        mma_f16_ts(to, r, lo, idesc, 1);
                    } else if (k == 0) {
                        mma_f16_ts_shifted<kLoBits>(to, r, hi, idesc);
                    } else {
                        mma_f16_ts(to, r, hi, idesc, 1);
                    }
                }
            };
            wait_one(&full[c % C::kStages], c / C::kStages);
            fence_proxy_async_smem();      // K and Q were written by threads, the MMAs read through the async proxy
#pragma unroll
            for (int b = 0; b < C::kBatches; ++b) {
                wait_one(&s_ready[b], c);
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int k = b; k < DK / 16; k += C::kBatches) state_low(k, 0);
                    if (b == C::kBatches - 1) {
                        state_high(0);
                        mma_commit(&made[0]);
                    }
                }
                __syncwarp();
            }
            wait_one(&o_done, c);      // the outputs have read their halves of D1 and D2
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < DK / 16; ++k) state_low(k, 1);
                state_high(1);
            }
            __syncwarp();
            wait_one(&r_ready, c);
            tc_fence_after();
            if (elect_one()) {
                row_product(0);
                mma_commit(&made[1]);
                row_product(1);
                mma_commit(&made[3]);
            }
            __syncwarp();
            wait_one(&w_ready, c);
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_f16_ts(tmem + C::kD3, tmem + C::kD2 + k * 16 + 8, kt + k * 128, kIdescT, 1);
                mma_f16_ts_shifted<kLoBits>(tmem + C::kD3, tmem + C::kD2, kt, kIdescT);
#pragma unroll
                for (int k = 1; k < 4; ++k) mma_f16_ts(tmem + C::kD3, tmem + C::kD2 + k * 16, kt + k * 128, kIdescT, 1);
                mma_commit(&made[2]);
                mma_commit(&empty[c % C::kStages]);
            }
            __syncwarp();
        }
        // every MMA has ended before its operands and tensor memory go
        if (chunks_here > 0) wait_one(&made[2], chunks_here - 1);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 23) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

int64_t chunk_slots(int64_t tokens, int64_t batch) { return tokens / kChunk + batch; }

template <int DK, int NG>
int launch_scan(const DeltaArgs& a, const Chunk* chunks, cudaStream_t stream) {
    using C = Scan<DK, NG>;
    static std::atomic<uint64_t> done{0};
    const int st = allow_smem(scan_kernel<DK, NG>, C::kSmem, done);
    if (st) return st;
    return launch(scan_kernel<DK, NG>, dim3((a.dv / 16 + NG - 1) / NG, a.v_heads, a.batch), dim3(C::kThreads), C::kSmem,
                  stream, a, chunks);
}

template <int DK>
int run_chunked(const DeltaArgs& a, void* workspace, cudaStream_t stream) {
    Chunk* chunks = static_cast<Chunk*>(workspace);
    constexpr int kSmem = ChunkSmem<DK>::kBytes;
    static std::atomic<uint64_t> done{0};
    int st = allow_smem(chunk_kernel<DK>, kSmem, done);
    if (st) return st;
    st = launch(chunk_kernel<DK>, dim3(static_cast<unsigned>(chunk_slots(a.tokens, a.batch)), a.v_heads), dim3(128),
                    kSmem, stream, a, chunks);
    if (st) return st;
    // The walk that takes the least time: rounds of blocks on the SMs, at 1.4 us a chunk with one column group a block,
    // 2.3 with two, 3.1 with whole heads.  Heads of 128 keys, all three forced:
    //   16 of 128 values, 8000 tokens: 210, 326, 427 us;  32 of 128, 8000: 408, 358, 460;  64 of 128, 4000: 413, 365, 273;
    //   2000 tokens, 200 of 16: 199, 258, 315;  140 of 32: 167, 155, 182;  200 of 32: 242, 261, 315;  80 of 64: 181, 200, 152.
    const int64_t heads = static_cast<int64_t>(a.batch) * a.v_heads;
    const int sms = sm_count();
    auto rounds = [&](int cols) { return (heads * ((a.dv + cols - 1) / cols) + sms - 1) / sms; };
    const int64_t single = 14 * rounds(16), pairs = 23 * rounds(32), whole = 31 * rounds(128);
    if (single <= pairs && single <= whole) return launch_scan<DK, 1>(a, chunks, stream);
    if (pairs <= whole) return launch_scan<DK, 2>(a, chunks, stream);
    static std::atomic<uint64_t> done_walk{0};
    if ((st = allow_smem(walk_kernel<DK>, Walk<DK>::kSmem, done_walk))) return st;
    return launch(walk_kernel<DK>, dim3((a.dv + 127) / 128, a.v_heads, a.batch), dim3(Walk<DK>::kThreads), Walk<DK>::kSmem, stream,
                  a, chunks);
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
    return run_step(a, args->key_dim, static_cast<cudaStream_t>(stream));
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
