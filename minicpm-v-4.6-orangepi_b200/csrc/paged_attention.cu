// Attention of one new token per sequence over a paged key-value cache:
//   o = softmax(scale q K^T) V,  lse = log sum exp(scale q K^T),
// with q_heads / kv_heads query heads sharing each key-value head.
//
// Bound by the cache's bytes (4 D bytes per key and kv head, read once).  The
// products run on the warp-level tensor MMA, not for their rate but because
// the fp32 FMAs of 8 query heads per key would take longer than the bytes do:
// per 16 keys and 256 dimensions a warp issues 48 MMAs, a fraction of the
// time in which its SM receives those 16 KB.
//
// Everything is transposed so that the few query heads are the MMA's n = 8:
// S^T (16 keys x 8 heads) = K Q^T, and O^T (D x 8 heads) = V^T P^T.  K comes
// as an A fragment through ldmatrix and V^T through its transposing form; S^T
// turns into the B fragment of the second product by an 8x8 register
// transpose.  P = 2^(s - max) is taken times 2^15 and split into hi + lo fp16 (the
// second MMA costs nothing here): weights down to 2^-18 of the maximum's keep 22 bits,
// smaller ones an absolute 2^-40 of it.  Without the factor fp16's end, 2^-24, would
// cut off the long tail behind one dominant key.  Scores, maxima, sums and outputs
// are fp32, the sums in the factor's scale too.
//
// Work is cut evenly however ragged the batch is: all (sequence, head group)
// rows' 16-key units form one line that is divided into one contiguous range
// per block.  Within its range the four warps of a block take every fourth
// unit, each through a ring of its own in shared memory that runs ahead
// across row ends; page numbers are looked up two units ahead of the copies.
// At a row's end the block joins its warps' (max, sum, O).  A row that
// lies in one block's range is written at once; of a row cut over several
// blocks every block leaves a partial result, and the last one to arrive
// joins them in order (kFan at a time, level by level, which bounds what one
// block has to read), so results do not depend on timing.
#include "mixing.cuh"

#include <cfloat>

namespace mcv {
unsigned take_attention_device_error();

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kUnit = 16;      // keys of a unit
constexpr int kFan = 16;       // partial results joined at a time
constexpr int kLevels = 3;     // levels of joining: kFan^3 blocks at most
constexpr int kMaxBatch = 4096;
constexpr int kMinUnits = 4;   // least units of a block: one per warp
constexpr float kPLog2 = 15.0f, kPInv = 1.0f / 32768.0f;   // probabilities and their sums are kept times 2^15, below fp16's 65504

static __device__ unsigned g_attention_dev_error;

template <int D>
struct Tile {
    static constexpr int kStages = 3;
    static constexpr int kRowBytes = D * 2;
    static constexpr int kStageBytes = 2 * kUnit * kRowBytes;           // K rows, then V rows
    static constexpr int kRingBytes = kStages * kStageBytes;            // per warp
    static constexpr int kJoinRow = D + 4;                              // floats; spreads the heads over the banks
    static constexpr int kJoinBytes = kWarps * 8 * kJoinRow * 4;
    static constexpr int kSmem = kWarps * kRingBytes + kJoinBytes + 2 * kWarps * 8 * 4;
    // With two tiles of query heads and D = 256 a thread's 255 registers do not hold queries and accumulators, and 360
    // bytes a thread are spilled; that kernel still reads the cache at 77 % of the copy rate (16 over 2 heads, 131071 keys).
    static constexpr int kBlocksPerSm = D == 256 ? 1 : (D == 128 ? 2 : 3);
};

struct AttnArgs {
    const __half* q;
    const __half* k;
    const __half* v;
    const int32_t* table;
    const int32_t* lengths;
    __half* out;
    float* lse;
    float* part;
    unsigned* counters;   // [kLevels][2 * grid]
    int64_t q_bs, q_hs, table_cols;
    uint32_t page_vecs;      // 16-byte vectors from page to page
    int batch, q_heads, kv_heads, group, head_groups, splits_of_group, num_pages, max_keys;
    float scale_log2;
    FastDiv page;
};

__device__ __forceinline__ int key_count(const AttnArgs& a, int b) {
    const int n = a.lengths[b];
    return n < 0 ? 0 : (n > a.max_keys ? a.max_keys : n);
}
__device__ __forceinline__ int units_of(int keys) { return (keys + kUnit - 1) / kUnit; }

// A row of the work line: one sequence and one group of query heads.
struct Row {
    int begin;       // first unit
    int b, hg, keys, units;
    __device__ __forceinline__ void next(const AttnArgs& a) {
        begin += units;
        if (++hg < a.head_groups) return;
        hg = 0;
        do {
            ++b;
            keys = b < a.batch ? key_count(a, b) : 0;
        } while (b < a.batch && keys == 0);
        units = units_of(keys);
    }
};

__device__ __forceinline__ float scale_of(float m, float top) { return m == -INFINITY ? 0.0f : exp2f(m - top); }

template <int D, int NT>
struct Part {
    static constexpr int kHeads = 8 * NT;
    static constexpr int kFloats = kHeads * (D + 2);
    float* p;
    __device__ __forceinline__ Part(float* base, int64_t slot) : p(base + slot * kFloats) {}
    __device__ __forceinline__ float* m() const { return p; }
    __device__ __forceinline__ float* l() const { return p + kHeads; }
    __device__ __forceinline__ float* o(int head) const { return p + 2 * kHeads + head * D; }
};

// Counts this block in at *counter (after its global writes); true in the
// last of `expected`, which leaves the counter at zero.  The barriers and the
// acquire-release addition order all threads' writes before it and all
// reads after it, on both sides.
__device__ __forceinline__ bool arrive_last(unsigned* counter, unsigned expected, int* flag) {
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned before;
        asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
        if (before == expected - 1) *counter = 0;
        *flag = before == expected - 1;
    }
    __syncthreads();
    return *flag != 0;
}

// Joins `n` <= kFan partial results (slot_of(0..n-1), in order).  to_out: normalised
// into the output rows; else back into slot_of(0).  `stats` (kFan + 1 rows of
// heads, shared memory) holds the maxima, then the weights.  Eight results'
// elements are in flight at once per thread (four with 16 heads of 256).
template <int D, int NT, typename SlotOf>
__device__ __forceinline__ void join_parts(const AttnArgs& a, int n, SlotOf slot_of, bool to_out, int b, int head0,
                                           int heads, float2* stats) {
    using P = Part<D, NT>;
    constexpr int kVec = D / 4;
    constexpr int kItems = (P::kHeads * kVec) / kThreads;
    constexpr int kRounds = kFan * P::kHeads / kThreads;
    constexpr int kBatch = kItems > 4 ? 4 : 8;
    float4 acc[kItems], o[kBatch][kItems];
    float sum[kItems];
    auto fetch = [&](int s0) {
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
            const float4* src = reinterpret_cast<const float4*>(P(a.part, slot_of(min(s0 + s, n - 1))).o(0)) + threadIdx.x;
#pragma unroll
            for (int i = 0; i < kItems; ++i)
                // heads of a group that ends before the tile were never written
                o[s][i] = s0 + s < n && (static_cast<int>(threadIdx.x) + i * kThreads) / kVec < heads
                              ? __ldcg(src + i * kThreads)
                              : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    };
    float m[kRounds], l[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const int i = threadIdx.x + r * kThreads, s = i / P::kHeads, h = i % P::kHeads;
        const P p(a.part, slot_of(min(s, n - 1)));
        const bool there = s < n && h < heads;
        m[r] = there ? __ldcg(p.m() + h) : -INFINITY;
        l[r] = there ? __ldcg(p.l() + h) : 0.0f;
    }
    fetch(0);
#pragma unroll
    for (int r = 0; r < kRounds; ++r) stats[threadIdx.x + r * kThreads].x = m[r];
    __syncthreads();
    float top[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const int h = threadIdx.x % P::kHeads;
        top[r] = -INFINITY;
#pragma unroll
        for (int s = 0; s < kFan; ++s) top[r] = fmaxf(top[r], stats[s * P::kHeads + h].x);
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const float w = scale_of(m[r], top[r]);
        stats[threadIdx.x + r * kThreads] = make_float2(w, w * l[r]);
        if (r == 0 && threadIdx.x < P::kHeads) stats[kFan * P::kHeads + threadIdx.x].x = top[r];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        sum[i] = 0.0f;
    }
#pragma unroll 1
    for (int s0 = 0;;) {
#pragma unroll
        for (int s = 0; s < kBatch; ++s)
#pragma unroll
            for (int i = 0; i < kItems; ++i) {
                // weights behind the last result are zero
                const float2 w = stats[(s0 + s) * P::kHeads + (threadIdx.x + i * kThreads) / kVec];
                sum[i] += w.y;
                acc[i].x += w.x * o[s][i].x;
                acc[i].y += w.x * o[s][i].y;
                acc[i].z += w.x * o[s][i].z;
                acc[i].w += w.x * o[s][i].w;
            }
        s0 += kBatch;
        if (s0 >= n) break;
        fetch(s0);
    }
    const P first(a.part, slot_of(0));
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int item = threadIdx.x + i * kThreads;
        const int h = item / kVec, d = (item % kVec) * 4;
        if (h >= heads) continue;
        const float2 all = make_float2(stats[kFan * P::kHeads + h].x, sum[i]);
        if (to_out) {
            const int64_t row = static_cast<int64_t>(b) * a.q_heads + head0 + h;
            const float inv = 1.0f / all.y;
            *reinterpret_cast<uint2*>(a.out + row * D + d) =
                make_uint2(h2_as_u32(__floats2half2_rn(acc[i].x * inv, acc[i].y * inv)),
                           h2_as_u32(__floats2half2_rn(acc[i].z * inv, acc[i].w * inv)));
            if (d == 0 && a.lse) a.lse[row] = (all.x + log2f(all.y * kPInv)) * 0.6931471805599453f;
        } else {
            // each element of slot_of(0) is read and written by one thread alone, and
            // its maxima and sums were read by all before the barriers above
            *reinterpret_cast<float4*>(first.o(h) + d) = acc[i];
            if (d == 0) {
                first.m()[h] = all.x;
                first.l()[h] = all.y;
            }
        }
    }
}

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, Tile<D>::kBlocksPerSm) attention_kernel(const AttnArgs a) {
    using T = Tile<D>;
    using P = Part<D, NT>;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int2 sums[kWarps], first;
    __shared__ int flag;
    float* join = reinterpret_cast<float*>(smem + kWarps * T::kRingBytes);
    float* join_m = join + kWarps * 8 * T::kJoinRow;
    float* join_l = join_m + kWarps * 8;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    pdl_trigger();
    pdl_wait();

    // sequences without keys: their rows are zero, with an empty sum
    auto empty_rows = [&]() {
        for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
            const int n = a.lengths[b];
            if (n > a.max_keys && tid == 0) atomicOr(&g_attention_dev_error, kDevErrIndex);
            if (n > 0) continue;
            const int64_t row = static_cast<int64_t>(b) * a.q_heads;
            uint4* o = reinterpret_cast<uint4*>(a.out + row * D);
            for (int i = tid; i < a.q_heads * (D / 8); i += kThreads) o[i] = make_uint4(0, 0, 0, 0);
            if (a.lse)
                for (int i = tid; i < a.q_heads; i += kThreads) a.lse[row + i] = -INFINITY;
        }
    };

    // ---- this block's range of the work line and the row that it begins in ----
    // Thread i counts a few sequences; up to 32, every warp counts them all by itself.
    const bool few = a.batch <= 32;
    const int per_thread = few ? 1 : (a.batch + kThreads - 1) / kThreads;
    const int b0 = (few ? lane : tid) * per_thread, b1 = min(b0 + per_thread, a.batch);
    int units = 0, rows = 0;
    for (int b = b0; b < b1; ++b) {
        const int n = units_of(key_count(a, b));
        units += n;
        rows += n > 0;
    }
    int total = __reduce_add_sync(0xffffffffu, units) * a.head_groups;
    int total_rows = __reduce_add_sync(0xffffffffu, rows) * a.head_groups;
    if (!few) {
        if (lane == 0) sums[warp] = make_int2(total, total_rows);
        __syncthreads();
        total = total_rows = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            total += sums[w].x;
            total_rows += sums[w].y;
        }
        __syncthreads();
    }
    // Ranges of the line are even, but a block whose range crosses a row's end joins
    // two rows, which a short call waits for.  With few rows each is divided by
    // itself: with total / (blocks - rows) units a block there are blocks enough, since
    // sum ceil(n_r / p) <= total / p + rows.  Taken where it costs a block at most
    // 128 KB more than the even ranges, total rows / (blocks (blocks - rows)) units:
    // joining twice was seen to take as long as 4 us, that many bytes' time.
    const int grid = gridDim.x, spare = grid - total_rows;
    const bool by_row = spare > 0 && static_cast<int64_t>(total) * total_rows * D <= static_cast<int64_t>(grid) * spare * 2048;
    const int div = by_row ? spare : grid;
    const int per = max(kMinUnits, (total + div - 1) / div);     // units of a block
    // what a sequence takes of the line: its units, or its blocks
    auto weight = [&](int b) {
        const int n = units_of(key_count(a, b));
        return a.head_groups * (by_row ? (n + per - 1) / per : n);
    };
    int mine = units * a.head_groups;
    if (by_row) {
        mine = 0;
        for (int b = b0; b < b1; ++b) mine += weight(b);
    }
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += u;
    }
    if (few) {
        total = __shfl_sync(0xffffffffu, before, 31);
    } else {
        if (lane == 31) sums[warp].x = before;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += sums[w].x;
            total += sums[w].x;
        }
    }
    before -= mine;
    int start = by_row ? blockIdx.x : min(static_cast<int64_t>(per) * blockIdx.x, static_cast<int64_t>(total));
    if (start >= total) {
        empty_rows();
        return;
    }
    int end = by_row ? 0 : min(static_cast<int64_t>(start) + per, static_cast<int64_t>(total));
    const bool owner = start >= before && start < before + mine;
    int row_b = b0;
    if (owner) {
        for (;; ++row_b) {
            const int n = weight(row_b);
            if (start < before + n) break;
            before += n;
        }
    }
    if (few) {
        const int from = __ffs(__ballot_sync(0xffffffffu, owner)) - 1;
        row_b = __shfl_sync(0xffffffffu, row_b, from);
        before = __shfl_sync(0xffffffffu, before, from);
    } else {
        if (owner) first = make_int2(row_b, before);
        __syncthreads();
        row_b = first.x;
        before = first.y;
    }
    Row row;
    row.b = row_b;
    row.keys = key_count(a, row.b);
    row.units = units_of(row.keys);
    int row_part = 0, row_parts = 0;      // by_row: this block's share of its row
    if (by_row) {
        const int blocks = (row.units + per - 1) / per;
        const int at = start - before;
        row.hg = at / blocks;
        row_part = at - row.hg * blocks;
        const int share = (row.units + blocks - 1) / blocks;
        row_parts = (row.units + share - 1) / share;
        row.begin = 0;
        start = row_part * share;
        end = min(start + share, row.units);
        if (start >= end) {
            empty_rows();
            return;
        }
    } else {
        row.hg = (start - before) / row.units;
        row.begin = before + row.hg * row.units;
    }

    // ---- the ring's producer side: the same lanes, running ahead ----
    constexpr int kVecs = D / 8;     // 16-byte vectors of a row
    const uint32_t ring = smem_u32(smem) + warp * T::kRingBytes;
    Row ahead = row;
    int u_look = start + warp, u_ahead = u_look;
    constexpr uint32_t kNone = 0xffffffffu;
    struct Look {          // row r of a unit, in lanes r and r + 16
        uint32_t at;       // place within the page in 16-byte vectors, kNone: no such row
        int page;
    };
    auto look_up = [&]() {
        Look x{kNone, 0};
        const int u = u_look;
        u_look += kWarps;
        if (u >= end) return x;
        while (u >= ahead.begin + ahead.units) ahead.next(a);
        const int key = (u - ahead.begin) * kUnit + (lane & 15);
        if (key >= ahead.keys) return x;
        const uint32_t page = a.page.div(key);
        x.page = a.table[ahead.b * a.table_cols + page];
        const int kvh = ahead.hg / a.splits_of_group;
        x.at = (kvh * a.page.d + (key - page * a.page.d)) * kVecs;
        return x;
    };
    auto issue = [&](int stage, const Look& x) {
        if (u_ahead < end) {
            const uint32_t base = ring + stage * T::kStageBytes;
            uint32_t src = kNone;      // the row's first vector in k and v
            if (x.at != kNone) {
                if (x.page >= 0 && x.page < a.num_pages) src = x.page * a.page_vecs + x.at;
                else atomicOr(&g_attention_dev_error, kDevErrIndex);
            }
#pragma unroll
            for (int i = 0; i < kUnit * kVecs / 32; ++i) {
                const int item = i * 32 + lane;
                const int r = item / kVecs, c = item % kVecs;
                const uint32_t off = __shfl_sync(0xffffffffu, src, r);
                const bool take = off != kNone;
                const uint64_t bytes = static_cast<uint64_t>(take ? off + c : 0) * 16;
                const uint32_t dst = base + r * T::kRowBytes + ((c ^ (r & 7)) << 4);
                cp_async16_or_zero(dst, reinterpret_cast<const char*>(a.k) + bytes, take);
                cp_async16_or_zero(dst + kUnit * T::kRowBytes, reinterpret_cast<const char*>(a.v) + bytes, take);
            }
        }
        cp_async_commit();
        u_ahead += kWarps;
    };

    // Q^T as B fragments: lane (g, t) holds head g, dims 2t, 2t+1 (+8) of each 16
    uint32_t qf[NT][D / 16][2];
    auto load_q = [&](const Row& r) {
        const int in_group = (r.hg % a.splits_of_group) * P::kHeads;
        const int head0 = (r.hg / a.splits_of_group) * a.group + in_group;
        const int heads = min(P::kHeads, a.group - in_group);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int h = n * 8 + g;
            const uint32_t* qr = reinterpret_cast<const uint32_t*>(a.q + r.b * a.q_bs + (head0 + (h < heads ? h : 0)) * a.q_hs);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
                qf[n][kk][0] = h < heads ? qr[kk * 8 + t] : 0u;
                qf[n][kk][1] = h < heads ? qr[kk * 8 + 4 + t] : 0u;
            }
        }
    };
    // pages are looked up two units ahead of their copies, queries a row ahead
    Look look0 = look_up(), look1 = look_up();
    load_q(row);
#pragma unroll 1
    for (int s = 0; s < T::kStages - 1; ++s) {
        issue(s, look0);
        look0 = look1;
        look1 = look_up();
    }
    empty_rows();

    // ldmatrix row addresses of this lane, before the swizzle
    const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_vec = lane >> 4;
    const int v_row = (lane & 7) + (lane >> 4) * 8, v_vec = (lane >> 3) & 1;
    int stage = 0;
    int u = start + warp;
    for (int pos = start; pos < end;) {
        const int seg_end = min(row.begin + row.units, end);
        const int kvh = row.hg / a.splits_of_group;
        const int in_group = (row.hg % a.splits_of_group) * P::kHeads;
        const int head0 = kvh * a.group + in_group;
        const int heads = min(P::kHeads, a.group - in_group);

        float acc[NT][D / 16][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.0f;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.0f;
        }

        for (; u < seg_end; u += kWarps) {
            cp_async_wait<T::kStages - 2>();
            __syncwarp();   // the unit has landed, and every lane is done with the stage that is filled next
            issue(stage == 0 ? T::kStages - 1 : stage - 1, look0);
            look0 = look1;
            look1 = look_up();
            const uint32_t kb = ring + stage * T::kStageBytes;
            const uint32_t vb = kb + kUnit * T::kRowBytes;
            float s[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
            {
                // two accumulator chains: an MMA's latency is several issue slots
                float s2[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) s2[n][0] = s2[n][1] = s2[n][2] = s2[n][3] = 0.0f;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk) {
                    uint32_t f[4];
                    ldsm4(f, kb + k_row * T::kRowBytes + (((kk * 2 + k_vec) ^ (k_row & 7)) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma16816(kk & 1 ? s2[n] : s[n], f, qf[n][kk][0], qf[n][kk][1]);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[n][i] += s2[n][i];
            }
            const int key = (u - row.begin) * kUnit + g;
            const bool in0 = key < row.keys, in1 = key + 8 < row.keys;
            uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                // columns 2t, 2t+1 are heads; rows g, g+8 keys
                float top[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    s[n][c] = in0 ? s[n][c] * a.scale_log2 : -INFINITY;
                    s[n][2 + c] = in1 ? s[n][2 + c] * a.scale_log2 : -INFINITY;
                    float x = fmaxf(s[n][c], s[n][2 + c]);
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                    top[c] = fmaxf(m[n][c], x);
                }
                if (__any_sync(0xffffffffu, top[0] > m[n][0] || top[1] > m[n][1])) {
                    const float w0 = scale_of(m[n][0], top[0]), w1 = scale_of(m[n][1], top[1]);
                    l[n][0] *= w0;
                    l[n][1] *= w1;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        acc[n][i][0] *= w0;
                        acc[n][i][1] *= w1;
                        acc[n][i][2] *= w0;
                        acc[n][i][3] *= w1;
                    }
                    m[n][0] = top[0];
                    m[n][1] = top[1];
                }
                float p[4];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    // no number above -inf so far: nothing to weigh yet
                    const float base = m[n][c] == -INFINITY ? 0.0f : m[n][c];
                    p[c] = exp2f(s[n][c] - base + kPLog2);
                    p[2 + c] = exp2f(s[n][2 + c] - base + kPLog2);
                    l[n][c] += p[c] + p[2 + c];
                }
                uint32_t lo;
                split_f16(p[0], p[1], ph[n][0], lo);
                ph[n][0] = movm_t(ph[n][0]);
                pl[n][0] = movm_t(lo);
                split_f16(p[2], p[3], ph[n][1], lo);
                ph[n][1] = movm_t(ph[n][1]);
                pl[n][1] = movm_t(lo);
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                uint32_t f[4];
                ldsm4_t(f, vb + v_row * T::kRowBytes + (((i * 2 + v_vec) ^ (v_row & 7)) << 4));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma16816(acc[n][i], f, ph[n][0], ph[n][1]);
                    mma16816(acc[n][i], f, pl[n][0], pl[n][1]);
                }
            }
            stage = stage + 1 == T::kStages ? 0 : stage + 1;
        }

        Row next = row;
        if (seg_end < end) {
            next.next(a);
            load_q(next);
        }

        // ---- join the block's warps ----
        const bool whole = row.begin >= start && row.begin + row.units <= end;
        // the row's blocks are c0 .. c0 + parts - 1; a row that begins inside c0's range uses its second slot
        const int c0 = by_row ? static_cast<int>(blockIdx.x) - row_part : row.begin / per;
        const int parts = by_row ? row_parts : (row.begin + row.units - 1) / per - c0 + 1;
        const bool second = !by_row && row.begin != c0 * per;
        auto slot_of_block = [&](int c) { return 2 * c + (second && c == c0 ? 1 : 0); };
        const P mine_part(a.part, slot_of_block(blockIdx.x));
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n * 8 >= heads) break;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = l[n][c];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
                if (g == 0) {
                    join_m[warp * 8 + 2 * t + c] = m[n][c];
                    join_l[warp * 8 + 2 * t + c] = x;
                }
            }
            float* jw = join + warp * 8 * T::kJoinRow;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    jw[(2 * t + (e & 1)) * T::kJoinRow + i * 16 + g + (e >> 1) * 8] = acc[n][i][e];
            __syncthreads();
            for (int item = tid; item < 8 * (D / 4); item += kThreads) {
                const int h = item / (D / 4), d = (item % (D / 4)) * 4;
                if (n * 8 + h >= heads) break;
                float top = join_m[h];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) top = fmaxf(top, join_m[w * 8 + h]);
                float sum = 0.0f;
                float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float x = scale_of(join_m[w * 8 + h], top);
                    const float4 y = *reinterpret_cast<const float4*>(join + (w * 8 + h) * T::kJoinRow + d);
                    sum += x * join_l[w * 8 + h];
                    o.x += x * y.x;
                    o.y += x * y.y;
                    o.z += x * y.z;
                    o.w += x * y.w;
                }
                if (whole) {
                    const int64_t orow = static_cast<int64_t>(row.b) * a.q_heads + head0 + n * 8 + h;
                    const float inv = 1.0f / sum;
                    *reinterpret_cast<uint2*>(a.out + orow * D + d) =
                        make_uint2(h2_as_u32(__floats2half2_rn(o.x * inv, o.y * inv)),
                                   h2_as_u32(__floats2half2_rn(o.z * inv, o.w * inv)));
                    if (d == 0 && a.lse) a.lse[orow] = (top + log2f(sum * kPInv)) * 0.6931471805599453f;
                } else {
                    *reinterpret_cast<float4*>(mine_part.o(n * 8 + h) + d) = o;
                    if (d == 0) {
                        mine_part.m()[n * 8 + h] = top;
                        mine_part.l()[n * 8 + h] = sum;
                    }
                }
            }
            __syncthreads();
        }
        if (!whole) {
            // kFan neighbours' results become one, kFan of those the next, ... each time by the last to arrive
            unsigned* counters = a.counters;
            for (int step = 1;; step *= kFan, counters += 2 * gridDim.x) {
                const int f0 = c0 + (static_cast<int>(blockIdx.x) - c0) / (step * kFan) * (step * kFan);
                const int n = min(kFan, (c0 + parts - f0 + step - 1) / step);
                if (!arrive_last(counters + slot_of_block(f0), n, &flag)) break;
                const bool all = step * kFan >= parts;
                join_parts<D, NT>(a, n, [&](int i) { return slot_of_block(f0 + i * step); }, all, row.b, head0, heads,
                                  reinterpret_cast<float2*>(join));
                if (all) break;
            }
            __syncthreads();   // join is written again
        }
        pos = seg_end;
        row = next;
    }
}

// Query heads of one group are served by ceil(group / (8 NT)) rows; NT = 2
// from 9 heads on, so that the cache is read once up to 16.
int tiles_for(int64_t group) { return group <= 8 ? 1 : 2; }

int blocks_per_sm(int64_t dim) { return dim == 256 ? 1 : (dim == 128 ? 2 : 3); }

// The counters come first and take the same room for every head size, so that
// calls of different shapes can share one workspace.
size_t counter_count() { return static_cast<size_t>(sm_count()) * 3 * 2 * kLevels; }

size_t part_floats(int64_t dim, int nt) { return static_cast<size_t>(8 * nt) * (dim + 2); }

size_t workspace_bytes_for(int64_t dim, int nt) {
    const size_t grid = static_cast<size_t>(sm_count()) * blocks_per_sm(dim);
    return counter_count() * sizeof(unsigned) + 2 * grid * part_floats(dim, nt) * sizeof(float);
}

template <int D, int NT>
int launch_attention(const AttnArgs& a, int grid, cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    const int st = allow_smem(attention_kernel<D, NT>, Tile<D>::kSmem, done);
    if (st) return st;
    return launch(attention_kernel<D, NT>, dim3(grid), dim3(kThreads), Tile<D>::kSmem, stream, a);
}

}  // namespace

unsigned take_attention_device_error() {
    unsigned v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_attention_dev_error, sizeof(v)) != cudaSuccess) return ~0u;
    if (v) cudaMemcpyToSymbol(g_attention_dev_error, &zero, sizeof(zero));
    return v;
}

}  // namespace mcv

using namespace mcv;

extern "C" {

size_t mcv_paged_attention_workspace_size(int64_t q_heads, int64_t kv_heads, int64_t head_dim) {
    if (q_heads < 1 || kv_heads < 1 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
    return workspace_bytes_for(head_dim, tiles_for(q_heads / kv_heads));
}

int mcv_paged_attention_decode(const mcv_rows* q, const mcv_kv_cache* cache, const void* page_table,
                               int64_t table_cols, const void* lengths, void* out, void* lse, int64_t batch,
                               int64_t q_heads, float scale, void* workspace, size_t workspace_bytes,
                               mcv_stream_t stream) {
    int st = check_kv_cache("paged_attention_decode", cache);
    if (st) return st;
    const int64_t dim = cache->head_dim;
    if (dim != 64 && dim != 128 && dim != 256)
        return fail(MCV_ERR_SHAPE, "paged_attention_decode: head_dim must be 64, 128 or 256");
    if ((st = check_rows("paged_attention_decode", "q", q, q_heads, dim))) return st;
    if (!page_table || !lengths || !out) return fail(MCV_ERR_NULL, "paged_attention_decode: null pointer");
    if (!aligned16(out)) return fail(MCV_ERR_ALIGN, "paged_attention_decode: out must be 16-byte aligned");
    if (batch < 1 || batch > kMaxBatch) return fail(MCV_ERR_SHAPE, "paged_attention_decode: batch must be 1..4096");
    if (q_heads < 1 || q_heads > 4096 || q_heads % cache->kv_heads)
        return fail(MCV_ERR_SHAPE, "paged_attention_decode: q_heads must be a multiple of the cache's kv_heads");
    if (table_cols < 1 || table_cols * cache->page_size > 0x7fffffffLL - kUnit || table_cols > 0x7fffffffLL)
        return fail(MCV_ERR_SHAPE, "paged_attention_decode: a sequence holds fewer than 2^31 - 16 keys");
    if (!(scale > 0.0f) || scale > FLT_MAX) return fail(MCV_ERR_VALUE, "paged_attention_decode: scale must be positive");
    const int64_t group = q_heads / cache->kv_heads;
    const int nt = tiles_for(group);
    if (!workspace || workspace_bytes < workspace_bytes_for(dim, nt))
        return fail(MCV_ERR_WORKSPACE, "paged_attention_decode: workspace missing or too small");
    if (!aligned16(workspace)) return fail(MCV_ERR_ALIGN, "paged_attention_decode: workspace must be 16-byte aligned");

    const int sms = sm_count();
    const int64_t splits = (group + 8 * nt - 1) / (8 * nt);
    const int64_t max_keys = table_cols * cache->page_size;
    const int64_t most = batch * cache->kv_heads * splits * ((max_keys + kUnit - 1) / kUnit);
    if (most > 0x7fffffffLL - kMinUnits)
        return fail(MCV_ERR_SHAPE, "paged_attention_decode: batch x kv heads x table capacity / 16 must stay below 2^31");
    if (static_cast<uint64_t>(cache->num_pages) * static_cast<uint64_t>(cache->page_stride / 8) >= 0xffffffffull)
        return fail(MCV_ERR_SHAPE, "paged_attention_decode: k and v may span 64 GB each");
    const int64_t want = (most + kMinUnits - 1) / kMinUnits;
    const int full = sms * blocks_per_sm(dim);
    const int grid = static_cast<int>(want < full ? want : full);

    AttnArgs a{static_cast<const __half*>(q->data), static_cast<const __half*>(cache->k),
               static_cast<const __half*>(cache->v), static_cast<const int32_t*>(page_table),
               static_cast<const int32_t*>(lengths), static_cast<__half*>(out), static_cast<float*>(lse), nullptr, nullptr,
               q->token_stride, q->head_stride, table_cols, static_cast<uint32_t>(cache->page_stride / 8), static_cast<int>(batch),
               static_cast<int>(q_heads), cache->kv_heads, static_cast<int>(group),
               static_cast<int>(cache->kv_heads * splits), static_cast<int>(splits), cache->num_pages,
               static_cast<int>(max_keys), scale * 1.4426950408889634f, FastDiv(static_cast<uint32_t>(cache->page_size))};
    a.counters = static_cast<unsigned*>(workspace);
    a.part = reinterpret_cast<float*>(a.counters + counter_count());
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dim == 256) return nt == 1 ? launch_attention<256, 1>(a, grid, s) : launch_attention<256, 2>(a, grid, s);
    if (dim == 128) return nt == 1 ? launch_attention<128, 1>(a, grid, s) : launch_attention<128, 2>(a, grid, s);
    return nt == 1 ? launch_attention<64, 1>(a, grid, s) : launch_attention<64, 2>(a, grid, s);
}

}  // extern "C"
