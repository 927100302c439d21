// Matrix product of 8-bit integers on the 5th-generation tensor cores:
//   C[m, n] = (sum_k A[m, k] W[n, k]) * a_scale[m] * w_scale[n]      A [M, K], W [N, K] int8, the sum in 32-bit integers
// and, gated, C[m, i] = silu(C'[m, 2i]) * C'[m, 2i + 1] over weight rows that alternate gate and up.  The sums are exact (|code| <= 128 and
// K < 131,072 keep them below 2^31), so a token's result depends neither on how K is cut nor on the batch it is in, to the last bit.
//
// Both operands are K-major; TMA brings 128-byte-swizzled tiles (128 codes a row) into a ring of shared-memory stages, one elected thread issues
// tcgen05.mma.kind::i8 (32 codes of K an instruction), the accumulators lie in tensor memory.  The weights sit in the instruction's M slot, the
// tokens in its N slot.  Two kernels, of which the one of the least expected time runs (choose below):
//   few tokens (gemm_int8_few_kernel): up to 128 weight rows x 16, 32, 64 or 128 tokens a block, two blocks an SM; K may be cut over a cluster of
//     2, 4 or 8 blocks, which add their integer tiles through distributed shared memory: no scratch, no flags, one launch;
//   many tokens (gemm_int8_pair_kernel): 256 weight rows x up to 256 tokens on pairs of blocks, persistent, the accumulator double-buffered.
// The scales are read through pointers without __restrict__, as an earlier kernel may have written them: loads of a const __restrict__ parameter may be moved ahead of
// the wait for it.
// Tails: rows beyond M or N and the end of K are zero-filled by TMA, stores are predicated.  Any K; the rows of A and of W lie a multiple of 16 bytes
// apart.  No cluster multicast is used.
//
// Measured (replayed from a graph for some milliseconds at 1,965 MHz, weights cycled past L2; in brackets the bytes at the measured copy rate of 6,547 GB/s, or the
// operations at 3,279 TOP/s, twice the measured bfloat16 rate: a yardstick, not a bound of the integer pipe): 1 x 6,144 x 4,096 5.9 us (3.9), 8 x 24,576 x 4,096
// gated 17.3 (15.4), 64 x 4,096 x 12,288 13.1 (7.9): the first bytes' way and a microsecond behind the last ones; 300 x 4,096 x 4,096 10.9 (3.1) and
// 300 x 4,096 x 12,288 23.7 (9.2): too few tiles to fill the device without low ones, and K walked whole; 2,048 x 6,144 x 4,096 36.7 (31.4: 2.6 rounds of tiles
// where 3 are paid), 4,096 x 24,576 x 4,096 gated 244 (251).  Under lasting load the clock falls: the last two take 42.5 us at 1,597 MHz and 282 at 1,327.
//
// The reference has no integer product (its own are half precision: spymaster2h/spyinfer src/backends/cuda/cublas/sgemm.cu:37-55).
#include <cuda.h>
#include <math.h>

#include "common.cuh"
#include "tcgen05.cuh"

SPY_MODULE(spy_gemm_int8)

namespace {

using namespace tc;

constexpr int BM = 128;            // weight rows of a block = the instruction's M (half of it on pairs)
constexpr int BK = 128;            // codes of K a stage = bytes of a swizzled row
constexpr int UMMA_K = 32;
// warp 0: TMA, warp 1: MMA and tensor memory, warps 2 and on: epilogue, in fours (each of four reads its own quarter of the tensor-memory lanes), the fours
// taking the tokens in turns.  Four warps alone read a tile of 128 tokens out in 3.1 us, eight in 1.6, and nothing runs beside that behind a block's last tile.
__host__ __device__ constexpr int epilogue_warps(int tokens) { return tokens >= 64 ? 8 : 4; }
__host__ __device__ constexpr int block_threads(int tokens) { return 64 + 32 * epilogue_warps(tokens); }
constexpr int MAX_K = 131071;
constexpr int MAX_ROWS = 1 << 22;  // of weights: the grid's second dimension at 64 a block; coordinates and tile numbers stay far inside 32 bits

// Instruction descriptor of kind::i8: signed 8-bit operands, both K-major, a 32-bit integer accumulator.
__device__ __forceinline__ uint32_t instr_desc_s8(int m, int n)
{
    uint32_t d = 0;
    d |= 2u << 4;                      // accumulator S32
    d |= 1u << 7;                      // A signed 8-bit
    d |= 1u << 10;                     // B signed 8-bit
    d |= (uint32_t)(n >> 3) << 17;
    d |= (uint32_t)(m >> 4) << 24;
    return d;
}
__device__ __forceinline__ void umma_s8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void umma_s8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// silu(g) * u = g u / (1 + exp(-g)) for a bfloat16 result.  Below zero it is formed as g exp(g) / (1 + exp(g)): the fast division gives 0 for divisors from
// 2^126 on, which 1 + exp(-g) is from g = -87.3 down, where a large u still makes a number of it.  The fast exponential is off by about 2 + 1.2 |g| ulp and the
// division by 2, together below 2^-16 of the result, far inside its rounding; from g = -87.3 down exp(g) is a subnormal number, and the result off by 2^-142 u.
__device__ __forceinline__ float silu_mul(float g, float u)
{
    const float e = __expf(-fabsf(g));
    return __fdividef(g < 0.f ? g * e : g, 1.0f + e) * u;
}

// One lane of a warp that has come together, always the same.
__device__ __forceinline__ bool elect_one()
{
    uint32_t chosen;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
    return chosen != 0;
}
template <int WARPS> __device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory"); }
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_shared_of(uint32_t cluster_addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d)
{
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

constexpr int TURN_LD = 36;                                  // floats between the tokens of a warp's chunk of some tokens x 32 weight rows
__host__ __device__ constexpr int turn_bytes(int cols) { return (cols * TURN_LD + 32) * 4; }   // and the tokens' scales

// Finishes COLS tokens of 32 weight rows: this lane holds weight row x0 + lane of the tokens from y on.  `turn` is the warp's own place in shared
// memory, where the numbers are turned so that the results leave in rows of 16 bytes a lane.
template <int COLS, typename TC, bool GATED>
__device__ __forceinline__ void store_chunk(TC* __restrict__ out, long long ld, int lane, int x0, int y, int x_end, int y_end, const uint32_t (&r)[COLS], float sw,
                                            float sa_lane, float* turn)
{
    const int count = min(COLS, y_end - y), outs = min(32, x_end - x0);
    if (outs <= 0 || count <= 0) return;      // the same for the whole warp
    float* sa = turn + COLS * TURN_LD;
    sa[lane] = sa_lane;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < COLS; j += 4) {
        const float4 s = *reinterpret_cast<const float4*>(sa + j);
        turn[j * TURN_LD + lane] = (float)(int)r[j] * s.x * sw;
        turn[(j + 1) * TURN_LD + lane] = (float)(int)r[j + 1] * s.y * sw;
        turn[(j + 2) * TURN_LD + lane] = (float)(int)r[j + 2] * s.z * sw;
        turn[(j + 3) * TURN_LD + lane] = (float)(int)r[j + 3] * s.w * sw;
    }
    __syncwarp();
    constexpr int PER = GATED ? 16 : 32;      // results of a token
    TC* dst = out + (size_t)y * ld + (GATED ? x0 / 2 : x0);
    if (outs == 32 && ld * (long long)sizeof(TC) % 16 == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
        if constexpr (GATED) {
            // two lanes a token, eight results each
            const int part = lane & 1;
#pragma unroll
            for (int i = 0; i < COLS / 16; ++i) {
                const int t = i * 16 + (lane >> 1);
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 v = *reinterpret_cast<const float4*>(turn + t * TURN_LD + part * 16 + 4 * e);
                    w[e] = pack_bf16(silu_mul(v.x, v.y), silu_mul(v.z, v.w));
                }
                if (t < count) *reinterpret_cast<uint4*>(dst + (size_t)t * ld + part * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else if constexpr (sizeof(TC) == 2) {
            // four lanes a token, eight results each
            const int part = lane & 3;
#pragma unroll
            for (int i = 0; i < COLS / 8; ++i) {
                const int t = i * 8 + (lane >> 2);
                const float4 v = *reinterpret_cast<const float4*>(turn + t * TURN_LD + part * 8);
                const float4 w = *reinterpret_cast<const float4*>(turn + t * TURN_LD + part * 8 + 4);
                if (t < count)
                    *reinterpret_cast<uint4*>(dst + (size_t)t * ld + part * 8) =
                        make_uint4(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w), pack_bf16(w.x, w.y), pack_bf16(w.z, w.w));
            }
        } else {
            const int part = lane & 7;
#pragma unroll
            for (int i = 0; i < COLS / 4; ++i) {
                const int t = i * 4 + (lane >> 3);
                if (t < count) *reinterpret_cast<float4*>(dst + (size_t)t * ld + part * 4) = *reinterpret_cast<const float4*>(turn + t * TURN_LD + part * 4);
            }
        }
    } else {
        const int results = GATED ? outs / 2 : outs;
        for (int i = lane; i < count * PER; i += 32) {
            const int t = i / PER, c = i % PER;
            if (c < results) {
                if constexpr (GATED) dst[(size_t)t * ld + c] = from_f32<TC>(silu_mul(turn[t * TURN_LD + 2 * c], turn[t * TURN_LD + 2 * c + 1]));
                else dst[(size_t)t * ld + c] = from_f32<TC>(turn[t * TURN_LD + c]);
            }
        }
    }
    __syncwarp();   // the next chunk's numbers may come
}

// ---- few tokens ------------------------------------------------------------------------------------------------------------------
// Two blocks share an SM, each with AREA bytes of stages.  A tile of fewer than 128 weight rows takes only its own bytes (rounded up to the
// swizzle's 1 KB); the tensor core still reads 128 rows: the spare ones come from whatever lies behind (the area ends with room for that) and feed
// accumulator rows that are never stored.
// What follows the last load is as short as it can be (3 us of 8 when the blocks of a cluster fetched one another's sums, 1 now): the scales are fetched while the tiles stream in; with K whole, each
// warp turns its rows in the ring, which is free by then, and stores them.  With K cut, block r of the cluster finishes the r-th part of the weight
// rows: every block writes its integer sums of these rows straight into block r's shared memory (`mail`, [source][group of four tokens][row]), one cluster barrier, and
// block r adds them up.  Up to 32 tokens the mail has a place of its own; beyond, it takes the ring's, and the blocks first tell one another that theirs is free.
template <int BN> struct Tile {
    static constexpr int Y_BYTES = BN * BK;
    static constexpr int TMEM_COLS = BN < 32 ? 32 : BN;
    static constexpr int COLS = BN < 32 ? BN : 32;              // tokens of a chunk that a warp reads out at a time
    static constexpr int WARPS = epilogue_warps(BN);
    static constexpr int THREADS = block_threads(BN);
    static constexpr int MAIL = BN * BM * 4;
    static constexpr bool MAIL_IN_RING = BN > 32;
    static constexpr int AREA = 110 * 1024 - (MAIL_IN_RING ? 0 : MAIL);
    static constexpr int MAX_STAGES = 12;
    static constexpr size_t SMEM = 110 * 1024 + 1024 /* alignment slack */ + 256 /* barriers */ + BN * 4 /* the tokens' scales */;
    __host__ __device__ static constexpr int x_bytes(int tile_rows) { return (tile_rows * BK + 1023) & ~1023; }
    __host__ __device__ static constexpr int stages(int tile_rows)
    {
        const int n = (AREA - (BM * BK - x_bytes(tile_rows))) / (x_bytes(tile_rows) + Y_BYTES);
        return n < MAX_STAGES ? n : MAX_STAGES;
    }
    static_assert(MAIL <= AREA && WARPS * turn_bytes(COLS) <= AREA, "what follows the main loop fits the ring");
};

// The end of a tile whose K is cut: this thread adds up weight row x of every STEP-th group of four tokens.  Gated: lanes 2i and 2i + 1 hold gate and
// up; of four tokens the even lane finishes the first two and the odd lane the others.
template <int SPLITS, int BN, typename TC, bool GATED>
__device__ __forceinline__ void finish_cut(TC* __restrict__ out, long long ld, const int4* mail, const float* sa, float sw, int x, int x_end, int y0, int tokens,
                                           int tid, int lane)
{
    constexpr int SHARE = BM / SPLITS, STEP = 32 * epilogue_warps(BN) / SHARE;      // groups of four tokens that the block finishes at a time
    const int4* got = mail + tid % SHARE;
    const bool inside = x < x_end, odd = (lane & 1) != 0;
    TC* dst = out + (size_t)y0 * ld + (GATED ? x / 2 : x);
#pragma unroll 2
    for (int q0 = 0; q0 < BN / 4; q0 += STEP) {
        const int q = q0 + tid / SHARE;
        if (4 * q0 >= tokens) break;                  // the same for the whole block
        int4 sum = make_int4(0, 0, 0, 0);
        float4 s4 = make_float4(0.f, 0.f, 0.f, 0.f);
        if (4 * q < tokens) {
            s4 = *reinterpret_cast<const float4*>(sa + 4 * q);
#pragma unroll
            for (int s = 0; s < SPLITS; ++s) {
                const int4 v = got[(s * (BN / 4) + q) * SHARE];
                sum.x += v.x;
                sum.y += v.y;
                sum.z += v.z;
                sum.w += v.w;
            }
        }
        const float v[4] = {(float)sum.x * s4.x * sw, (float)sum.y * s4.y * sw, (float)sum.z * s4.z * sw, (float)sum.w * s4.w * sw};
        if constexpr (GATED) {
            const float p = __shfl_xor_sync(0xffffffffu, odd ? v[0] : v[2], 1), r = __shfl_xor_sync(0xffffffffu, odd ? v[1] : v[3], 1);
            const float first = odd ? silu_mul(p, v[2]) : silu_mul(v[0], p), second = odd ? silu_mul(r, v[3]) : silu_mul(v[1], r);
            const int t = 4 * q + (odd ? 2 : 0);
            if (inside && t < tokens) dst[(size_t)t * ld] = from_f32<TC>(first);
            if (inside && t + 1 < tokens) dst[(size_t)(t + 1) * ld] = from_f32<TC>(second);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (inside && 4 * q + e < tokens) dst[(size_t)(4 * q + e) * ld] = from_f32<TC>(v[e]);
        }
    }
}

// Block (token tile, K range) = (blockIdx.x / splits, blockIdx.x % splits) of weight tile blockIdx.y; the K ranges of a tile are a cluster.
template <int BN, typename TC, bool GATED>
__global__ void __launch_bounds__(block_threads(BN), 2)
gemm_int8_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const float* w_scale,
                     const float* a_scale, TC* __restrict__ out, long long ld, int N, int M, int k_blocks, int splits, int tile_rows, int settled,
                     int* status, const uint8_t* __restrict__ next_weights, long long next_bytes)
{
    using T = Tile<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    int4* mail = reinterpret_cast<int4*>(T::MAIL_IN_RING ? tiles : tiles + T::AREA);
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(tiles + 110 * 1024);
    uint64_t* empty_bar = full_bar + T::MAX_STAGES;
    uint64_t* accum_bar = empty_bar + T::MAX_STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accum_bar + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* sa = reinterpret_cast<float*>(tiles + 110 * 1024 + 256);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % splits;                       // the block's place in its cluster
    const int x0 = blockIdx.y * tile_rows, y0 = blockIdx.x / splits * BN;
    const int kb0 = (int)((long long)rank * k_blocks / splits), num_kb = (int)((long long)(rank + 1) * k_blocks / splits) - kb0;
    const uint32_t stage_tx = (uint32_t)tile_rows * BK + T::Y_BYTES;
    const int x_bytes = T::x_bytes(tile_rows), stage_bytes = x_bytes + T::Y_BYTES, stages = T::stages(tile_rows);

    if (threadIdx.x == 0) {
#pragma unroll 1
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar + s, 1);
            mbar_init(empty_bar + s, 1);
        }
        mbar_init(accum_bar, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(tmem_slot, T::TMEM_COLS);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    pdl_launch_dependents();
    // the cluster's first barrier: a block's mail may be written.  All but the warps that free the ring arrive here.
    if (splits > 1 && (!T::MAIL_IN_RING || warp < 2)) cluster_arrive();
    if (warp == 0) {
        // The whole warp walks the loops of this role and the next, and one lane of it requests and issues: what the instructions take is then the same for
        // the warp, not a lane's (a block's K block of 128 codes, 16 tokens: 0.32 us with all of it on one lane, 0.22 now).
        const bool lead = elect_one();
        // settled weights depend on no earlier kernel: their tiles for the first stages are requested before the wait for the kernels ahead in the stream
        if (!settled) pdl_wait();
        const int pre = min(num_kb, stages);
#pragma unroll 1
        for (int i = 0; i < pre; ++i) {
            if (lead) {
                mbar_expect_tx(full_bar + i, stage_tx);
                tma_load_2d(smem_u32(tiles + (size_t)i * stage_bytes), &map_w, (kb0 + i) * BK, x0, full_bar + i);
            }
        }
        pdl_wait();
#pragma unroll 1
        for (int i = 0; i < pre; ++i)
            if (lead) tma_load_2d(smem_u32(tiles + (size_t)i * stage_bytes + x_bytes), &map_a, (kb0 + i) * BK, y0, full_bar + i);
        int s = 0;
        uint32_t phase = 1;   // of the round before: the first wait on a stage is for its first release
#pragma unroll 1
        for (int i = pre; i < num_kb; ++i) {
            if (!__all_sync(0xffffffffu, mbar_wait(empty_bar + s, phase ^ 1, abort_flag))) break;
            if (lead) {
                uint8_t* xs = tiles + (size_t)s * stage_bytes;
                mbar_expect_tx(full_bar + s, stage_tx);
                tma_load_2d(smem_u32(xs), &map_w, (kb0 + i) * BK, x0, full_bar + s);
                tma_load_2d(smem_u32(xs + x_bytes), &map_a, (kb0 + i) * BK, y0, full_bar + s);
            }
            if (++s == stages) {
                s = 0;
                phase ^= 1;
            }
        }
        // Every load of this block has been requested: what follows in a decode step are short kernels that leave the memory idle, and then a product
        // whose weights are known now.  This block asks for its share of them to be brought into L2 meanwhile.  A hint only: nothing waits for it.
        if (lead && next_bytes > 0) {
            const long long blocks = (long long)gridDim.x * gridDim.y, me = blockIdx.x + (long long)gridDim.x * blockIdx.y;
            const long long piece = ((next_bytes + blocks - 1) / blocks + 127) / 128 * 128;
            const long long stop = min(next_bytes, (me + 1) * piece);
#pragma unroll 1
            for (long long at = me * piece; at < stop; at += 16384) l2_prefetch(next_weights + at, (uint32_t)(min(stop - at, 16384LL) & ~15LL));
        }
    } else if (warp == 1) {
        const bool lead = elect_one();
        const uint32_t idesc = instr_desc_s8(BM, BN);
        const uint64_t dx0 = desc_k_major(smem_u32(tiles)), dy0 = desc_k_major(smem_u32(tiles + x_bytes));
        const uint32_t step = (uint32_t)stage_bytes >> 4, end = step * stages;
        int s = 0;
        uint32_t phase = 0, at = 0;           // at: where the stage lies, in the descriptors' units
        pdl_wait();                           // the limit of the waits below is not for the kernels ahead
#pragma unroll 1
        for (int i = 0; i < num_kb; ++i) {
            if (!__all_sync(0xffffffffu, mbar_wait(full_bar + s, phase, abort_flag))) break;
            fence_after_sync();
            if (lead) {
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k) {
                    const uint32_t adv = at + (uint32_t)((k * UMMA_K) >> 4);
                    umma_s8(tmem_base, dx0 + adv, dy0 + adv, idesc, (i > 0 || k > 0) ? 1u : 0u);
                }
                umma_commit(empty_bar + s);   // the stage is free again when these MMAs have read it
            }
            ++s;
            at += step;
            if (at == end) {
                s = 0;
                at = 0;
                phase ^= 1;
            }
        }
        if (lead) umma_commit(accum_bar);     // the accumulator is complete when every MMA has finished
    } else {
        // warp w reads tensor-memory lanes 32 (w % 4) .. + 31, i.e. weight rows of the tile
        const int quarter = warp & 3, turns = (warp - 2) >> 2, row = quarter * 32 + lane, tid = threadIdx.x - 64;
        const int tokens = min(BN, M - y0), x_end = min(N, x0 + tile_rows);
        const int share = BM / splits, part = rank * share + (tid & (share - 1));        // K cut: the weight row that this thread finishes
        const int x = x0 + (splits > 1 ? part : row);
        float sw = settled && x < x_end ? w_scale[x] : 0.f;
        pdl_wait();                           // the tokens' scales and the output belong to kernels ahead in the stream until here
        if (!settled && x < x_end) sw = w_scale[x];
        if (tid < BN) sa[tid] = tid < tokens ? a_scale[y0 + tid] : 0.f;
        epilogue_barrier<T::WARPS>();
        // one lane asks for the warp: lanes that left the wait one by one would meet the warp-wide loads and barriers behind it apart
        const bool ok = mbar_wait_warp(accum_bar, 0, abort_flag);
        __syncwarp();
        fence_after_sync();
        const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16);
        constexpr int COLS = T::COLS, STEP = COLS * (T::WARPS / 4);
        if (splits == 1) {
            float* turn = reinterpret_cast<float*>(tiles + (warp - 2) * turn_bytes(COLS));
#pragma unroll 1
            for (int c = turns * COLS; c < tokens && ok; c += STEP) {
                uint32_t r[COLS];
                tmem_load<COLS>(acc + (uint32_t)c, r);
                tmem_wait_ld(r);
                store_chunk<COLS, TC, GATED>(out, ld, lane, x0 + quarter * 32, y0 + c, x_end, M, r, sw, lane < COLS ? sa[c + lane] : 0.f, turn);
            }
        } else {
            if constexpr (T::MAIL_IN_RING) cluster_arrive();
            cluster_wait();
            const uint32_t to = map_to_rank(smem_u32(mail + (size_t)rank * (BN / 4) * share + (row & (share - 1))), row / share);
#pragma unroll 1
            for (int c = turns * COLS; c < tokens && ok; c += STEP) {
                uint32_t r[COLS];
                tmem_load<COLS>(acc + (uint32_t)c, r);
                tmem_wait_ld(r);
#pragma unroll
                for (int j = 0; j < COLS; j += 4)
                    if (c + j < tokens) store_shared_of(to + (uint32_t)((c + j) / 4 * share) * 16, r[j], r[j + 1], r[j + 2], r[j + 3]);
            }
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            if (ok) {
                if (splits == 2) finish_cut<2, BN, TC, GATED>(out, ld, mail, sa, sw, x0 + part, x_end, y0, tokens, tid, lane);
                else if (splits == 4) finish_cut<4, BN, TC, GATED>(out, ld, mail, sa, sw, x0 + part, x_end, y0, tokens, tid, lane);
                else finish_cut<8, BN, TC, GATED>(out, ld, mail, sa, sw, x0 + part, x_end, y0, tokens, tid, lane);
            }
        }
    }
    __syncwarp();                             // the lanes that had no part in a role wait for the one that had
    fence_before_sync();
    if (splits > 1 && warp < 2) {
        cluster_wait();
        cluster_arrive();
        cluster_wait();
    }

    __syncthreads();
    if (*abort_flag) {
        // a wait ran out: copies that may still be in flight get time to land before the shared memory is released, then it is reported
        if (threadIdx.x == 0) {
            const unsigned long long t0 = global_timer();
            while (global_timer() - t0 < 2000000ull) { }
            report_status(status, SPY_STATUS_WAIT_TIMEOUT, (int)(blockIdx.x + blockIdx.y * gridDim.x));
        }
        __syncthreads();
    }
    if (warp == 1) {
        fence_after_sync();
        tmem_dealloc(tmem_base, T::TMEM_COLS);
    }
}

// ---- many tokens -----------------------------------------------------------------------------------------------------------------
// A cluster of two blocks on neighbouring SMs computes one tile of 256 weight rows and up to 256 tokens: each block loads its 128 weight rows and its
// half of the tile's tokens, the leader (rank 0) issues tcgen05.mma.cta_group::2 instructions that read both blocks' shared memory and
// accumulate each block's 128 rows in its own tensor memory; both blocks' epilogue warps read their halves back and turn them in shared memory
// on the way out.  The TMA loads of both blocks complete on the leader's full barrier; a commit frees a stage, and publishes an accumulator, in both
// blocks; the peer's epilogue threads arrive on the leader's accumulator-empty barrier.  Cluster c walks tiles c, c + clusters, ...; tiles are numbered
// with the token tiles fastest, so that clusters side by side share weight tiles in L2.

// The tokens in `count` tiles whose heights are multiples of 32 and differ by 32 at most: the first `tall` tiles have `rows` tokens, the others 32 fewer.
struct TokenTiles {
    int count, rows, tall;
    __host__ __device__ int first(int t) const { return t * rows - (t > tall ? (t - tall) * 32 : 0); }
    __host__ __device__ int height(int t) const { return t < tall ? rows : rows - 32; }
};
static inline TokenTiles token_tiles(int M, int count)
{
    TokenTiles t;
    const int runs = (M + 31) / 32, each = runs / count, more = runs % count;
    t.count = count;
    t.rows = 32 * (more > 0 ? each + 1 : each);
    t.tall = more > 0 ? more : count;
    return t;
}

constexpr int PAIR_BN = 256;                                 // tensor-memory columns of an accumulator
constexpr int PAIR_MAX_STAGES = 10;
constexpr int PAIR_X_BYTES = BM * BK;
constexpr int PAIR_AREA = 6 * 2 * PAIR_X_BYTES;              // the ring: six stages at 256 tokens a tile, more at fewer
constexpr int PAIR_COLS = 16;                                // tokens of a chunk that an epilogue warp reads out at a time
constexpr int PAIR_WARPS = epilogue_warps(PAIR_BN);
constexpr int PAIR_THREADS = block_threads(PAIR_BN);
constexpr size_t PAIR_SMEM = (size_t)PAIR_AREA + PAIR_WARPS * turn_bytes(PAIR_COLS) + 1024 /* alignment slack */ + 256 /* barriers */;
__host__ __device__ constexpr int pair_stage_bytes(int token_rows) { return PAIR_X_BYTES + token_rows / 2 * BK; }
__host__ __device__ constexpr int pair_stages(int token_rows)
{
    const int n = PAIR_AREA / pair_stage_bytes(token_rows);
    return n < PAIR_MAX_STAGES ? n : PAIR_MAX_STAGES;
}

template <typename TC, bool GATED>
__global__ void __launch_bounds__(PAIR_THREADS, 1)
gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const float* w_scale,
                      const float* a_scale, TC* __restrict__ out, long long ld, int N, int M, int k_blocks, TokenTiles tokens, int num_tiles,
                      int settled, int* status)
{
    const int stages = pair_stages(tokens.rows), stage_bytes = pair_stage_bytes(tokens.rows);   // a lower tile's copies bring spare rows behind its own
    extern __shared__ uint8_t smem_raw[];
    uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(tiles + PAIR_AREA + PAIR_WARPS * turn_bytes(PAIR_COLS));   // the leader's are used
    uint64_t* empty_bar = full_bar + PAIR_MAX_STAGES;   // every block's own
    uint64_t* acc_full = empty_bar + PAIR_MAX_STAGES;   // [2] every block's own
    uint64_t* acc_empty = acc_full + 2;                 // [2] the leader's are used: an arrival of every epilogue thread of both
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int cluster = blockIdx.x >> 1, clusters = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar + s, 1);
            mbar_init(empty_bar + s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full + b, 1);
            mbar_init(acc_empty + b, 2 * 32 * PAIR_WARPS);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    // The allocation is one for the pair.  Asked for before the other block runs it never comes back: without this barrier prompts of 640 tokens
    // through 36 layers, where a block's start can be held up by the many small blocks of a quantisation on its SM, stopped within some hundred steps.
    cluster_sync();   // both blocks run, and their barriers are initialised
    // settled weights' first stages are requested beside the allocation and before the wait for the kernels ahead in the stream
    const int pre = min(k_blocks, stages);
    const bool lead = elect_one();      // whole warps walk the loops, as in the kernel above (2,048 x 6,144 x 4,096: 41.5 us on one lane, 37 now)
    if (warp == 0) {
        const int x0 = (cluster / tokens.count) * (2 * BM) + (int)rank * BM;
        if (!settled) pdl_wait();
        if (lead) {
            for (int i = 0; i < pre; ++i) {
                if (rank == 0) mbar_expect_tx(full_bar + i, 2u * stage_bytes);     // both blocks' bytes
                tma_load_2d_pair(smem_u32(tiles + (size_t)i * stage_bytes), &map_w, i * BK, x0, map_to_rank(smem_u32(full_bar + i), 0));
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 2u * PAIR_BN);
    }
    fence_before_sync();
    cluster_sync();   // both blocks' tensor memory is allocated before it is used from the other side
    fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    pdl_launch_dependents();
    if (warp == 0) {
        pdl_wait();
        int s = pre == stages ? 0 : pre;
        uint32_t phase = pre == stages ? 1 : 0;   // of the ring's round; the first round's waits end at once
        bool ok = true;
        for (int tile = cluster; ok && tile < num_tiles; tile += clusters) {
            const int ty = tile % tokens.count;
            const int x0 = (tile / tokens.count) * (2 * BM) + (int)rank * BM, y0 = tokens.first(ty) + (int)rank * (tokens.height(ty) / 2);
            int kb = 0;
            if (tile == cluster) {
                for (; kb < pre; ++kb)
                    if (lead) tma_load_2d_pair(smem_u32(tiles + (size_t)kb * stage_bytes + PAIR_X_BYTES), &map_a, kb * BK, y0, map_to_rank(smem_u32(full_bar + kb), 0));
            }
#pragma unroll 1
            for (; kb < k_blocks; ++kb) {
                ok = __all_sync(0xffffffffu, mbar_wait(empty_bar + s, phase ^ 1, abort_flag));
                if (!ok) break;
                if (lead) {
                    uint8_t* xs = tiles + (size_t)s * stage_bytes;
                    if (rank == 0) mbar_expect_tx(full_bar + s, 2u * stage_bytes);
                    const uint32_t leader_full = map_to_rank(smem_u32(full_bar + s), 0);
                    tma_load_2d_pair(smem_u32(xs), &map_w, kb * BK, x0, leader_full);
                    tma_load_2d_pair(smem_u32(xs + PAIR_X_BYTES), &map_a, kb * BK, y0, leader_full);
                }
                if (++s == stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0) {
            const uint64_t dx0 = desc_k_major(smem_u32(tiles)), dy0 = desc_k_major(smem_u32(tiles + PAIR_X_BYTES));
            const uint32_t step = (uint32_t)stage_bytes >> 4, end = step * stages;
            int s = 0;
            uint32_t phase = 0, at = 0;       // at: where the stage lies, in the descriptors' units
            int i = 0;
            bool ok = true;
            pdl_wait();       // the limit of the waits below is not for the kernels ahead
            for (int tile = cluster; ok && tile < num_tiles; tile += clusters, ++i) {
                const uint32_t idesc = instr_desc_s8(2 * BM, tokens.height(tile % tokens.count));
                const int buf = i & 1;
                const uint32_t aph = (uint32_t)(i >> 1) & 1;
                if (i >= 2) ok = __all_sync(0xffffffffu, mbar_wait(acc_empty + buf, aph ^ 1, abort_flag));   // both blocks' epilogues have read this buffer's last tile
                if (!ok) break;
                fence_after_sync();
                const uint32_t acc = tmem_base + (uint32_t)buf * PAIR_BN;
#pragma unroll 1
                for (int kb = 0; kb < k_blocks; ++kb) {
                    ok = __all_sync(0xffffffffu, mbar_wait(full_bar + s, phase, abort_flag));
                    if (!ok) break;
                    fence_after_sync();
                    if (lead) {
#pragma unroll
                        for (int k = 0; k < BK / UMMA_K; ++k) {
                            const uint32_t adv = at + (uint32_t)((k * UMMA_K) >> 4);
                            umma_s8_pair(acc, dx0 + adv, dy0 + adv, idesc, (kb > 0 || k > 0) ? 1u : 0u);
                        }
                        umma_commit_pair(empty_bar + s);
                    }
                    ++s;
                    at += step;
                    if (at == end) {
                        s = 0;
                        at = 0;
                        phase ^= 1;
                    }
                }
                if (ok && lead) umma_commit_pair(acc_full + buf);
            }
        }
    } else {
        const int quarter = warp & 3, turns = (warp - 2) >> 2;
        float* turn = reinterpret_cast<float*>(tiles + PAIR_AREA + (warp - 2) * turn_bytes(PAIR_COLS));
        pdl_wait();   // the scales and the output belong to kernels ahead in the stream until here
        int i = 0;
        for (int tile = cluster; tile < num_tiles; tile += clusters, ++i) {
            const int buf = i & 1;
            const uint32_t aph = (uint32_t)(i >> 1) & 1;
            const int x0 = (tile / tokens.count) * (2 * BM) + (int)rank * BM + quarter * 32, ty = tile % tokens.count;   // the warp's first weight row
            const int y0 = tokens.first(ty), height = tokens.height(ty), y_end = min(M, y0 + height);
            const float sw = x0 + lane < N ? w_scale[x0 + lane] : 0.f;
            // the scales of a chunk's tokens, and the chunk itself, are requested a chunk ahead
            constexpr int STEP = PAIR_COLS * (PAIR_WARPS / 4);
            auto scale_of = [&](int c) { return lane < PAIR_COLS && y0 + c + lane < y_end ? a_scale[y0 + c + lane] : 0.f; };
            const uint32_t acc = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * PAIR_BN);
            int c = turns * PAIR_COLS;
            float sa = scale_of(c);
            const bool ok = mbar_wait_warp(acc_full + buf, aph, abort_flag);     // one lane asks: the warp goes on together
            __syncwarp();
            if (!ok) break;
            fence_after_sync();
            uint32_t ahead[PAIR_COLS];
            if (c < height) tmem_load<PAIR_COLS>(acc + (uint32_t)c, ahead);
#pragma unroll 1
            for (; c < height; c += STEP) {
                uint32_t r[PAIR_COLS];
                tmem_wait_ld(ahead);
#pragma unroll
                for (int j = 0; j < PAIR_COLS; ++j) r[j] = ahead[j];
                const float sa_now = sa;
                if (c + STEP < height) {
                    tmem_load<PAIR_COLS>(acc + (uint32_t)(c + STEP), ahead);
                    sa = scale_of(c + STEP);
                }
                store_chunk<PAIR_COLS, TC, GATED>(out, ld, lane, x0, y0 + c, N, y_end, r, sw, sa_now, turn);
            }
            fence_before_sync();
            if (rank == 0) mbar_arrive(acc_empty + buf);
            else mbar_arrive_cluster(map_to_rank(smem_u32(acc_empty + buf), 0));
        }
    }

    __syncwarp();     // the lanes that had no part in a role wait for the one that had
    fence_before_sync();
    __syncthreads();
    if (*abort_flag) {
        if (threadIdx.x == 0) {
            const unsigned long long t0 = global_timer();
            while (global_timer() - t0 < 2000000ull) { }
            report_status(status, SPY_STATUS_WAIT_TIMEOUT, (int)blockIdx.x);
        }
        __syncthreads();
    }
    cluster_sync();   // neither block leaves (and frees tensor memory the pair shares) while the other may still use it
    if (warp == 1) {
        fence_after_sync();
        tmem_dealloc_pair(tmem_base, 2u * PAIR_BN);
    }
}

// A [rows, K] matrix of codes with K contiguous; box = 128 codes x box_rows rows, 128-byte swizzle.
static int make_map(CUtensorMap* map, const void* ptr, long long rows, long long K, long long ld, int box_rows)
{
    EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) SPY_FAIL("gemm_int8: cuTensorMapEncodeTiled is not available from the driver");
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld};
    cuuint32_t box[2] = {(cuuint32_t)BK, (cuuint32_t)box_rows};
    cuuint32_t elem[2] = {1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) SPY_FAIL("gemm_int8: cuTensorMapEncodeTiled failed with code %d (rows %lld, K %lld, ld %lld)", (int)r, rows, K, ld);
    return 0;
}

// How a product is run.  pairs: `count` token tiles on pairs of blocks; else token tiles of `bn` on single blocks with tile_rows weight rows, K cut `splits` ways.
struct Plan {
    bool pairs;
    int count, bn, splits, tile_rows;
};

// The plan is the one of the least expected time, in us, with rates in bytes a us.  Both kernels: what is fixed, plus the slowest of what the main loop
// waits for, plus the read-out behind it.  The numbers were fitted to the measurements of 18 weight sizes (512 x 8,192 to 51,200 x 5,120) at 1 to 4,096
// tokens with all tiles and cuts: the chosen plans take 1.4 % longer than the fastest of all measured on average, 21 % at worst (5,003 x 2,055, 512 tokens).
// Which kernel, for instance (us, few / pairs): 6,144 x 4,096 at 128 tokens 10.7 / 11.5, 384 13.8 / 13.7; 34,816 x 5,120 gated at 64 tokens 29.5 / 31.8, 200
// 46.2 / 37.1.  How K is cut (1 / 2 / 4 / 8 ways, 8 tokens): 6,144 x 4,096 9.0 / 7.5 / 6.7 / 9.9, 4,096 x 12,288 22.7 / 14.1 / 11.3 / 10.7, 24,576 x 4,096
// 17.9 / 21.9 / 22.6 / -.
static double few_time(int M, int N, int k_blocks, int bn, int splits, int rows, int sms)
{
    const double blocks = (double)((M + bn - 1) / bn) * ((N + rows - 1) / rows) * splits, depth = (k_blocks + splits - 1) / splits;
    const double stage = (double)(rows + bn) * BK, tokens = (M < bn ? M : bn) / 128.0;
    const double even = blocks / sms, most = (double)(((long long)blocks + sms - 1) / sms);
    const double room = splits > 2 ? 1.85 * sms : 2.0 * sms;                          // clusters of 4 and 8 leave some SMs with one block
    const double per_sm = blocks <= room ? fmax(1.0, 0.61 * most + 0.39 * even) : 1.52 * even;      // an SM with one more; the last of many waves is not full
    double load = (double)N * k_blocks * BK / 1.2e7;                                  // the weights from memory; some come while what is fixed passes
    load = fmax(load, depth * fmax(0.22, stage / 8.3e4));                             // a block's stages, one after the other: issued, and fetched
    load = fmax(load, per_sm * depth * stage / 1.15e5);                               // an SM's
    const double cut = splits == 1 ? 0.0 : (splits == 2 ? 0.3 : (splits == 4 ? 0.6 : 0.9)) + 2.2 * tokens;      // the sums' way between blocks
    return 1.95 + cut + 1.8 * tokens + 0.25 * even + load;
}
static double pair_time(int M, int N, int k_blocks, int count, int sms)
{
    const TokenTiles t = token_tiles(M, count);
    const int clusters = sms / 2 > 0 ? sms / 2 : 1;
    const double height = t.rows / 256.0, rounds = (double)(((long long)((N + 2 * BM - 1) / (2 * BM)) * count + clusters - 1) / clusters);
    const double load = fmax((double)N * k_blocks * BK / 1.2e7, rounds * k_blocks * pair_stage_bytes(t.rows) / 1.12e5);
    return 6.2 + load + 2.2 * height + 1.8 * (rounds - 1) * height;
}

static Plan choose(int M, int N, int K, int sms)
{
    const int k_blocks = (K + BK - 1) / BK;
    const int tile = M <= 16 ? 16 : (M <= 32 ? 32 : (M <= 64 ? 64 : 128));
    Plan best = {false, 0, tile, 1, BM};
    double least = 1e30;
    for (int bn = tile; bn >= 16 && 2 * bn >= tile; bn /= 2) {
        for (int splits = 1; splits <= 8 && (splits == 1 || k_blocks >= 2 * splits); splits *= 2) {
            for (int rows = BM; rows >= (splits == 1 ? 64 : BM); rows -= 32) {      // weight rows of a multiple of what a warp reads out
                const double t = few_time(M, N, k_blocks, bn, splits, rows, sms);
                if (t < least && (N + rows - 1) / rows <= 65535) {       // the launch's limit
                    least = t;
                    best = {false, 0, bn, splits, rows};
                }
            }
        }
    }
    if (M < 64) return best;
    const int lowest = (M + 255) / 256, runs = (M + 31) / 32;
    for (int count = lowest; count <= runs && count <= 2 * lowest + 2 && count <= lowest + 16; ++count) {
        const double t = pair_time(M, N, k_blocks, count, sms);
        if (t < least) {
            least = t;
            best = {true, count, 0, 1, BM};
        }
    }
    return best;
}

template <int BN, typename TC, bool GATED>
static int launch_few(const Plan& p, const CUtensorMap& mw, const CUtensorMap& ma, const float* w_scale, const float* a_scale, void* C, long long ldc, int M,
                      int N, int k_blocks, int settled, int* status, cudaStream_t stream, const void* next_weights, long long next_bytes)
{
    using T = Tile<BN>;
    auto kernel = gemm_int8_few_kernel<BN, TC, GATED>;
    SPY_ONCE_PER_DEVICE {
        SPY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)T::SMEM));
    }
    const dim3 grid((unsigned)((M + BN - 1) / BN * p.splits), (unsigned)((N + p.tile_rows - 1) / p.tile_rows));
    if (p.splits == 1)
        spy_launch(kernel, grid, dim3(T::THREADS), T::SMEM, stream, mw, ma, w_scale, a_scale, (TC*)C, ldc, N, M, k_blocks, p.splits, p.tile_rows, settled,
                   status, (const uint8_t*)next_weights, next_bytes);
    else
        spy_launch_cluster(kernel, grid, dim3(T::THREADS), T::SMEM, stream, (unsigned)p.splits, mw, ma, w_scale, a_scale, (TC*)C, ldc, N, M, k_blocks,
                           p.splits, p.tile_rows, settled, status, (const uint8_t*)next_weights, next_bytes);
    SPY_CHECK_LAUNCH("gemm_int8");
    return 0;
}

template <typename TC, bool GATED>
static int launch_pairs(const Plan& p, const CUtensorMap& mw, const CUtensorMap& ma, const float* w_scale, const float* a_scale, void* C, long long ldc, int M,
                        int N, int k_blocks, const TokenTiles& tokens, int settled, int* status, cudaStream_t stream)
{
    auto kernel = gemm_int8_pair_kernel<TC, GATED>;
    static int clusters_of_device[SPY_MAX_DEVICES] = {};
    int& clusters_max = clusters_of_device[spy_device()];
    if (clusters_max == 0) {
        SPY_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)PAIR_SMEM));
        const int sms = spy_sm_count();
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(sms / 2 * 2);
        cfg.blockDim = dim3(PAIR_THREADS);
        cfg.dynamicSmemBytes = PAIR_SMEM;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int active = 0;
        SPY_CUDA(cudaOccupancyMaxActiveClusters(&active, kernel, &cfg));
        if (active <= 0) SPY_FAIL("gemm_int8: no cluster of two blocks fits the device");
        clusters_max = active < sms / 2 ? active : sms / 2;
    }
    const long long num_tiles = (long long)((N + 2 * BM - 1) / (2 * BM)) * tokens.count;
    if (num_tiles > 0x7fffffffLL) SPY_FAIL("gemm_int8: %lld tiles exceed the kernel's range", num_tiles);
    const int clusters = (int)(num_tiles < clusters_max ? num_tiles : clusters_max);
    spy_launch_cluster(kernel, dim3(2 * clusters), dim3(PAIR_THREADS), PAIR_SMEM, stream, 2u, mw, ma, w_scale, a_scale, (TC*)C, ldc, N, M, k_blocks, tokens,
                       (int)num_tiles, settled, status);
    SPY_CHECK_LAUNCH("gemm_int8 (pairs)");
    return 0;
}

template <typename TC, bool GATED>
static int run(const void* A, long long lda, const float* a_scale, const void* W, long long ldw, const float* w_scale, void* C, long long ldc, int M, int N,
               int K, int settled, int* status, cudaStream_t stream, const void* next_weights, long long next_bytes)
{
    const Plan p = choose(M, N, K, spy_sm_count());
    const int k_blocks = (K + BK - 1) / BK;
    CUtensorMap mw, ma;
    if (p.pairs) {
        const TokenTiles tokens = token_tiles(M, p.count);
        if (make_map(&mw, W, N, K, ldw, BM) || make_map(&ma, A, M, K, lda, tokens.rows / 2)) return 1;
        return launch_pairs<TC, GATED>(p, mw, ma, w_scale, a_scale, C, ldc, M, N, k_blocks, tokens, settled, status, stream);
    }
    if (make_map(&mw, W, N, K, ldw, p.tile_rows) || make_map(&ma, A, M, K, lda, p.bn)) return 1;
    if (p.bn == 16) return launch_few<16, TC, GATED>(p, mw, ma, w_scale, a_scale, C, ldc, M, N, k_blocks, settled, status, stream, next_weights, next_bytes);
    if (p.bn == 32) return launch_few<32, TC, GATED>(p, mw, ma, w_scale, a_scale, C, ldc, M, N, k_blocks, settled, status, stream, next_weights, next_bytes);
    if (p.bn == 64) return launch_few<64, TC, GATED>(p, mw, ma, w_scale, a_scale, C, ldc, M, N, k_blocks, settled, status, stream, next_weights, next_bytes);
    return launch_few<128, TC, GATED>(p, mw, ma, w_scale, a_scale, C, ldc, M, N, k_blocks, settled, status, stream, next_weights, next_bytes);
}

}  // namespace

// A [M, K] and W [N, K] int8, rows lda / ldw bytes apart (multiples of 16); a_scale [M], w_scale [N]; C [M, N] of c_dtype, rows ldc elements apart.
// gated: W's rows alternate gate and up rows, C is [M, N / 2] bfloat16.  status: null, or two ints that receive a code if a bounded wait runs out.
// settled: no kernel that may still run writes W or w_scale; they are then read ahead of the wait for the kernels before this one.
// next_weights / next_bytes (may be null / 0): memory that a later kernel of the stream will read, which the kernel for few tokens asks to be brought into L2.
extern "C" int spy_gemm_int8(const void* A, long long lda, const float* a_scale, const void* W, long long ldw, const float* w_scale, void* C, int c_dtype,
                             long long ldc, int M, int N, int K, int gated, int settled, int* status, cudaStream_t stream, const void* next_weights,
                             long long next_bytes)
{
    if (next_weights == nullptr || next_bytes <= 0 || (reinterpret_cast<uintptr_t>(next_weights) & 15)) {
        next_weights = nullptr;
        next_bytes = 0;
    }
    if (M <= 0 || N <= 0) return 0;
    if (M > MAX_ROWS || N > MAX_ROWS) SPY_FAIL("gemm_int8: %d x %d results: at most %d a side", M, N, MAX_ROWS);
    if (K <= 0 || K > MAX_K) SPY_FAIL("gemm_int8: K %d must lie in 1..%d (32-bit sums)", K, MAX_K);
    if (lda % 16 != 0 || ldw % 16 != 0) SPY_FAIL("gemm_int8: row distances %lld/%lld must be multiples of 16 bytes", lda, ldw);
    if ((reinterpret_cast<uintptr_t>(A) & 15) || (reinterpret_cast<uintptr_t>(W) & 15)) SPY_FAIL("gemm_int8: operands must be 16-byte aligned");
    if (gated && (N % 2 != 0 || c_dtype != SPY_BF16)) SPY_FAIL("gemm_int8: the gated epilogue needs an even N and bfloat16 output");
    if (gated) return run<bf16, true>(A, lda, a_scale, W, ldw, w_scale, C, ldc, M, N, K, settled, status, stream, next_weights, next_bytes);
    if (c_dtype == SPY_BF16) return run<bf16, false>(A, lda, a_scale, W, ldw, w_scale, C, ldc, M, N, K, settled, status, stream, next_weights, next_bytes);
    if (c_dtype == SPY_F32) return run<float, false>(A, lda, a_scale, W, ldw, w_scale, C, ldc, M, N, K, settled, status, stream, next_weights, next_bytes);
    SPY_FAIL("gemm_int8: unknown output dtype code %d", c_dtype);
}

// How a product of these sizes is run on a device of `sms` SMs; needs no device.  plan[5]: 1 on pairs of blocks; tokens of a tile (the tallest, on pairs);
// token tiles; ways that K is cut; weight rows of a tile.
extern "C" int spy_gemm_int8_plan(int M, int N, int K, int sms, int* plan)
{
    if (M <= 0 || M > MAX_ROWS || N <= 0 || N > MAX_ROWS || K <= 0 || K > MAX_K || sms <= 0) SPY_FAIL("gemm_int8: no plan for %d x %d x %d on %d SMs", M, N, K, sms);
    const Plan p = choose(M, N, K, sms);
    plan[0] = p.pairs ? 1 : 0;
    plan[1] = p.pairs ? token_tiles(M, p.count).rows : p.bn;
    plan[2] = p.pairs ? p.count : (M + p.bn - 1) / p.bn;
    plan[3] = p.splits;
    plan[4] = p.pairs ? 2 * BM : p.tile_rows;
    return 0;
}
