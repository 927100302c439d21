// Rows of 8-bit codes with one 32-bit scale each, made in one pass over the row:
//   quantize:  amax = max |x|,  code = the integer nearest 127 x / amax (ties to even),  scale = amax / 127
//   rms norm:  v = x[row] (+ delta[row], itself possibly a sum of split-K partial products), 32-bit sums, stored into x when write_back;
//              y = v * w rounded to 32 bits, quantised as above;  scale = amax / 127 / sqrt(mean(v^2) + eps)
// so that code * scale is the normed row: the factor 1 / sqrt(..) cancels in the codes and goes into the scale alone.
//
// The codes are exact: 127 y / amax is compared with the half between two integers without being rounded first.  In 32 bits
// t = y * (127 / amax) is off by at most |t| 2^-24 <= 7.6e-6 from the quotient (the fused multiply-add rounds t itself to the integer
// directly), so only where t lies within 2e-5 of a half is the question left open; there 254 y and (2 n + 1) amax are compared without rounding
// (one group of eight in 3,000 of float32 numbers; bfloat16 rows have exact halves, and one in sixty: those have a shorter way, encode8).  The codes depend on no summation order and on no
// approximation, and a test can ask for equality.
//
// A row of zeros has codes 0 and scale 0.  A row with a NaN or an infinity has codes 0 and the scale NaN: what is made of it is NaN, and no
// other row is touched.  |code| <= 127: -128 does not occur.  Squares that sum beyond the largest 32-bit number (values from 2^64 / sqrt(len) on) are summed
// once more of the row times 2^-80, so that finite rows have finite scales that are not 0 (rmsnorm.cu, with the same formula, gives zeros there).
//
// Rows of codes lie a multiple of 16 bytes apart (the product fetches them by TMA); bytes between a row's end and the next row are not written.
// What an earlier kernel may have written is read through pointers without __restrict__: of a const __restrict__ parameter the compiler takes it that nothing
// changes while the kernel runs, and then moves its loads ahead of the wait for the kernels before (pdl_wait), whose blocks this one's run beside.
// The outputs have it, which is enough for loads to pass stores.
//
// The reference keeps no 8-bit values anywhere (its weights are half precision: spymaster2h/spyinfer src/utils/safetensors_reader.cpp:101-122).
#include <math.h>

#include "common.cuh"

SPY_MODULE(spy_quant_int8)

namespace {

constexpr int STATUS_BAD_ROW = 5;      // beside the codes of common.cuh
constexpr float MAGIC = 12582912.0f;   // 1.5 * 2^23: added to a small number it leaves the nearest integer in the low bits

__device__ __forceinline__ void load8(const float* p, float (&v)[8])
{
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void load8(const bf16* p, float (&v)[8])
{
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8])
{
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16* p, const float (&v)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// The eight elements of a row that group g of this thread holds; what lies behind the end is zero.  WHOLE: rows of a multiple of 8 elements on
// 16-byte borders, a thread holds neighbours.  Else a warp's lanes hold neighbours, so that their plain loads and stores meet in few sectors.
template <bool WHOLE> __device__ __forceinline__ int place(int g, int e) { return WHOLE ? (g * blockDim.x + threadIdx.x) * 8 + e : (g * 8 + e) * blockDim.x + threadIdx.x; }
template <bool WHOLE, typename T> __device__ __forceinline__ void fetch(const T* row, int g, int len, float (&v)[8])
{
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if constexpr (WHOLE) {
        if (place<true>(g, 0) < len) load8(row + place<true>(g, 0), v);
    } else if constexpr (sizeof(T) == 2) {
        // as plain words, widened when all are on their way (1,531 x 4,999: one conversion a load 21.6 us)
        uint32_t raw[8] = {};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (place<false>(g, e) < len) raw[e] = reinterpret_cast<const unsigned short*>(row)[place<false>(g, e)];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(raw[e] << 16);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (place<false>(g, e) < len) v[e] = row[place<false>(g, e)];
    }
}
template <bool WHOLE, typename T> __device__ __forceinline__ void put(T* row, int g, int len, const float (&v)[8])
{
    if constexpr (WHOLE) {
        if (place<true>(g, 0) < len) store8(row + place<true>(g, 0), v);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (place<false>(g, e) < len) row[place<false>(g, e)] = from_f32<T>(v[e]);
    }
}

// The larger of m and |v|, NaN if either is: as bits, where a NaN is above the infinity and that above every number.
__device__ __forceinline__ uint32_t size_max(uint32_t m, float v) { return max(m, __float_as_uint(v) & 0x7fffffffu); }

// The whole number nearest to 127 y / amax, ties to even, by the sign of 254 y - (2 n + 1) amax with n the whole number below the quotient: hi + lo is
// the second product exactly, and near the half the fused difference to hi is exact as well (a few of the 31 bits of 254 y are left); elsewhere
// the sign is plain.
__device__ __forceinline__ int nearest_exact(float y, float k, float amax)
{
    const float n = floorf(y * k), b = 2.0f * n + 1.0f;
    const float hi = __fmul_rn(b, amax), lo = fmaf(b, amax, -hi), d = fmaf(254.0f, y, -hi);
    const int low = (int)n;
    return d > lo ? low + 1 : (d < lo ? low : low + (low & 1));
}

// The codes of eight numbers, four in a word.  k = 127 / amax.  BF16: the numbers and amax have 8 significant bits.  A quotient t is then a half or at least
// t / (254 * 255) away from one, 250 times what y * k is off by, so that only halves can come out on the wrong side, and 127 y - n amax is exact.
template <bool BF16> __device__ __forceinline__ uint2 encode8(const float (&y)[8], float k, float amax)
{
    // Numbers that are looked at together: of bfloat16 one warp in four has a half among 4 a lane, two in five among 8 (24,576 x 4,096 by 8 / 4 / 2: 50.8 / 49.4
    // / 53.7 us, with loads that ran ahead of the wait for the kernel before; 51.5 since they do not).
    constexpr int PART = BF16 ? 4 : 8;
    uint32_t m[8];
#pragma unroll
    for (int part = 0; part < 8; part += PART) {
        float far = 0.f;
#pragma unroll
        for (int e = part; e < part + PART; ++e) {
            const float n = fmaf(y[e], k, MAGIC);
            far = fmaxf(far, fabsf(fmaf(y[e], k, MAGIC - n)));
            m[e] = __float_as_uint(n);
        }
        if (far > 0.49998f) {
#pragma unroll
            for (int e = part; e < part + PART; ++e) {
                if constexpr (BF16) {
                    const float d = fmaf(MAGIC - __uint_as_float(m[e]), amax, 127.0f * y[e]);
                    if (fabsf(d) * 2.0f == amax && (m[e] & 1)) m[e] += d > 0.f ? 1u : 0xffffffffu;
                } else {
                    m[e] = (uint32_t)nearest_exact(y[e], k, amax);
                }
            }
        }
    }
    return make_uint2(__byte_perm(__byte_perm(m[0], m[1], 0x0040), __byte_perm(m[2], m[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(m[4], m[5], 0x0040), __byte_perm(m[6], m[7], 0x0040), 0x5410));
}
template <bool WHOLE> __device__ __forceinline__ void put_codes(int8_t* row, int g, int len, uint2 c)
{
    if constexpr (WHOLE) {
        if (place<true>(g, 0) < len) *reinterpret_cast<uint2*>(row + place<true>(g, 0)) = c;
    } else {
        // Four lanes hold four neighbours of each element: two exchanges give lane q of the four the neighbours of elements q and q + 4, which it stores as words.
        // The whole warp comes here.  1,531 x 4,999 float32: 12.6 us with the codes stored one by one, 9.3 in words (both with
        // loads that ran ahead of the wait for the kernel before; 9.8 since they do not).
        const int q = threadIdx.x & 3;
        const bool far = q >= 2, odd = (q & 1) != 0;
        uint32_t keep = __byte_perm(c.x, c.y, far ? 0x7632 : 0x5410);
        uint32_t got = __shfl_xor_sync(0xffffffffu, __byte_perm(c.x, c.y, far ? 0x5410 : 0x7632), 2);
        const uint32_t low = far ? got : keep, high = far ? keep : got;       // of the lower and the upper lane: two codes of the first word, two of the second
        keep = __byte_perm(low, high, odd ? 0x7351 : 0x6240);
        got = __shfl_xor_sync(0xffffffffu, __byte_perm(low, high, odd ? 0x6240 : 0x7351), 1);
        const uint32_t a = odd ? got : keep, b = odd ? keep : got;
        const uint32_t word[2] = {__byte_perm(a, b, 0x5140), __byte_perm(a, b, 0x7362)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = place<false>(g, q + 4 * h) - q;       // q is this thread's place in its four as well
            if (at + 4 <= len) {
                *reinterpret_cast<uint32_t*>(row + at) = word[h];
            } else {
#pragma unroll
                for (int i = 0; i < 3; ++i)
                    if (at + i < len) row[at + i] = (int8_t)(word[h] >> (8 * i));
            }
        }
    }
}

// What the codes of a row are formed with.  Rows below 2^-100 are lifted by 2^100 first, so that 127 / amax stays a number, and rows above 2^100
// lowered by 2^-30, so that 255 amax does (exact but for numbers far below half a code); a row of zeros, or with a NaN or an infinity in it, is
// replaced by zeros.
struct RowScale {
    float k, amax, lift;
    bool plain, none;
};
__device__ __forceinline__ RowScale row_scale(uint32_t size)
{
    RowScale s;
    s.none = size == 0 || size >= 0x7f800000u;
    s.amax = s.none ? 1.f : __uint_as_float(size);
    s.lift = s.amax < 0x1p-100f ? 0x1p100f : (s.amax > 0x1p100f ? 0x1p-30f : 1.f);
    s.plain = !s.none && s.lift == 1.f;
    s.amax *= s.lift;
    s.k = 127.0f / s.amax;
    return s;
}
__device__ __forceinline__ float scale_of(uint32_t size, float factor)
{
    return size >= 0x7f800000u ? __int_as_float(0x7fc00000) : __uint_as_float(size) / 127.0f * factor;
}
template <bool BF16> __device__ __forceinline__ uint2 encode_group(float (&y)[8], const RowScale& s)
{
    if (!s.plain) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = s.none ? 0.f : y[e] * s.lift;
    }
    return encode8<BF16>(y, s.k, s.amax);
}
template <bool WHOLE, int GROUPS, bool BF16 = false>
__device__ __forceinline__ void encode_row(int8_t* row, int len, float (&y)[GROUPS][8], uint32_t size)
{
    const RowScale s = row_scale(size);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) put_codes<WHOLE>(row, g, len, encode_group<BF16>(y[g], s));
}

// Sum and largest size over the block, one barrier; `part` holds 2 x 32 words and is used once a launch.
template <bool WITH_SUM> __device__ __forceinline__ void block_reduce(float& sum, uint32_t& size, uint32_t* part)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    size = __reduce_max_sync(0xffffffffu, size);
    if (WITH_SUM) sum = warp_sum(sum);
    if (lane == 0) {
        part[warp] = size;
        if (WITH_SUM) part[32 + warp] = __float_as_uint(sum);
    }
    __syncthreads();
    size = __reduce_max_sync(0xffffffffu, lane < warps ? part[lane] : 0u);
    if (WITH_SUM) sum = warp_sum(lane < warps ? __uint_as_float(part[32 + lane]) : 0.f);
}

// One more sum over the block behind block_reduce, through the same words.
__device__ __forceinline__ float block_sum_again(float sum, uint32_t* part)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    sum = warp_sum(sum);
    __syncthreads();          // every warp has read what block_reduce left
    if (lane == 0) part[warp] = __float_as_uint(sum);
    __syncthreads();
    return warp_sum(lane < warps ? __uint_as_float(part[lane]) : 0.f);
}

template <typename T, bool WHOLE, int GROUPS>
__global__ void __launch_bounds__(1024) quantize_kernel(const T* x, long long ldx, int8_t* __restrict__ codes, long long ldc,
                                                        float* __restrict__ scales, int len)
{
    __shared__ uint32_t part[32];
    pdl_enter();
    const T* row = x + (size_t)blockIdx.x * ldx;
    float v[GROUPS][8];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) fetch<WHOLE>(row, g, len, v[g]);
    uint32_t size = 0;
    float none = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int e = 0; e < 8; ++e) size = size_max(size, v[g][e]);
    block_reduce<false>(none, size, part);
    encode_row<WHOLE, GROUPS, sizeof(T) == 2>(codes + (size_t)blockIdx.x * ldc, len, v, size);
    if (threadIdx.x == 0) scales[blockIdx.x] = scale_of(size, 1.f);
}

// bfloat16 rows of whole groups: the row is kept as it was read, two elements in a register, and the largest size is taken of two at once.
template <int GROUPS>
__global__ void __launch_bounds__(1024) quantize_packed_kernel(const bf16* x, long long ldx, int8_t* __restrict__ codes, long long ldc,
                                                               float* __restrict__ scales, int len)
{
    __shared__ uint32_t part[32];
    pdl_enter();
    const bf16* row = x + (size_t)blockIdx.x * ldx;
    uint4 v[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        v[g] = make_uint4(0, 0, 0, 0);
        if (place<true>(g, 0) < len) v[g] = *reinterpret_cast<const uint4*>(row + place<true>(g, 0));
    }
    uint32_t two = 0;       // of bfloat16 bits without their signs the larger number is the larger size, a NaN the largest
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
        two = __vmaxu2(__vmaxu2(two, __vmaxu2(v[g].x & 0x7fff7fffu, v[g].y & 0x7fff7fffu)), __vmaxu2(v[g].z & 0x7fff7fffu, v[g].w & 0x7fff7fffu));
    uint32_t size = max(two << 16, two & 0xffff0000u);
    float none = 0.f;
    block_reduce<false>(none, size, part);
    const RowScale s = row_scale(size);
    int8_t* out = codes + (size_t)blockIdx.x * ldc;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        float y[8] = {__uint_as_float(v[g].x << 16), __uint_as_float(v[g].x & 0xffff0000u), __uint_as_float(v[g].y << 16), __uint_as_float(v[g].y & 0xffff0000u),
                      __uint_as_float(v[g].z << 16), __uint_as_float(v[g].z & 0xffff0000u), __uint_as_float(v[g].w << 16), __uint_as_float(v[g].w & 0xffff0000u)};
        put_codes<true>(out, g, len, encode_group<true>(y, s));
    }
    if (threadIdx.x == 0) scales[blockIdx.x] = scale_of(size, 1.f);
}

// Rows longer than a block holds: read once for the largest size and once more, from L2, for the codes.
template <typename T>
__global__ void __launch_bounds__(1024) quantize_long_kernel(const T* x, long long ldx, int8_t* __restrict__ codes, long long ldc,
                                                             float* __restrict__ scales, int len)
{
    __shared__ uint32_t part[32];
    pdl_enter();
    const T* row = x + (size_t)blockIdx.x * ldx;
    uint32_t size = 0;
    float none = 0.f;
    const int piece = blockDim.x * 8;
    for (int at = 0; len - at > 0; at += piece) {
        float v[8];
        fetch<false>(row + at, 0, len - at, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) size = size_max(size, v[e]);
        if (len - at <= piece) break;
    }
    block_reduce<false>(none, size, part);
    int8_t* out = codes + (size_t)blockIdx.x * ldc;
    for (int at = 0; len - at > 0; at += piece) {
        float v[1][8];
        fetch<false>(row + at, 0, len - at, v[0]);
        encode_row<false, 1, sizeof(T) == 2>(out + at, len - at, v, size);
        if (len - at <= piece) break;
    }
    if (threadIdx.x == 0) scales[blockIdx.x] = scale_of(size, 1.f);
}

template <typename TX, typename TD, typename TW, bool WHOLE, int GROUPS>
__global__ void __launch_bounds__(1024) rmsnorm_int8_kernel(TX* x, const TD* delta, int splits, long long split_stride, const int* rows,
                                                            const TW* w, int8_t* __restrict__ codes, long long ldc,
                                                            float* __restrict__ scales, int total, int len, float eps, int write_back, int settled, int* status)
{
    __shared__ uint32_t part[64];
    pdl_launch_dependents();
    // a settled weight depends on no kernel ahead in the stream: it is loaded before the wait for them (a row of 4,096: 2.1 us, behind it 2.4)
    float w_first[8];
    if constexpr (GROUPS == 1) {
        if (settled) fetch<WHOLE>(w, 0, len, w_first);
    }
    pdl_wait();
    if constexpr (GROUPS == 1) {
        if (!settled) fetch<WHOLE>(w, 0, len, w_first);
    }
    int src = blockIdx.x;
    if (rows) src = rows[blockIdx.x];
    if (rows && (src < 0 || src >= total)) {         // no row of x: nothing is read, the result is not a number
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) put_codes<WHOLE>(codes + (size_t)blockIdx.x * ldc, g, len, make_uint2(0, 0));
        if (threadIdx.x == 0) {
            scales[blockIdx.x] = __int_as_float(0x7fc00000);
            report_status(status, STATUS_BAD_ROW, blockIdx.x);
        }
        return;
    }
    TX* xr = x + (size_t)src * len;
    const TD* dr = delta ? delta + (size_t)src * len : nullptr;
    float v[GROUPS][8];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) fetch<WHOLE>(xr, g, len, v[g]);
    for (int s = 0; s < splits; ++s) {       // the partial products are added in their order
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            float d[8];
            fetch<WHOLE>(dr + (size_t)s * split_stride, g, len, d);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[g][e] = __fadd_rn(v[g][e], d[e]);
        }
    }
    if (write_back) {        // all of it ahead of the weight's loads, which may not pass a store to x
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) put<WHOLE>(xr, g, len, v[g]);
    }
    float ss = 0.f, low = 0.f;       // low: this thread's sum times 2^-160, formed where the sum itself has become infinite
    uint32_t size = 0;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        float wv[8];
        if constexpr (GROUPS > 1) fetch<WHOLE>(w, g, len, wv);
        const float before = ss;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += v[g][e] * v[g][e];
        if (ss == INFINITY) {
            if (before < INFINITY) low = before * 0x1p-80f * 0x1p-80f;
#pragma unroll
            for (int e = 0; e < 8; ++e) low += (v[g][e] * 0x1p-80f) * (v[g][e] * 0x1p-80f);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[g][e] = __fmul_rn(v[g][e], GROUPS > 1 ? wv[e] : w_first[e]);
            size = size_max(size, v[g][e]);
        }
    }
    if (ss < INFINITY) low = ss * 0x1p-80f * 0x1p-80f;
    block_reduce<true>(ss, size, part);
    encode_row<WHOLE, GROUPS>(codes + (size_t)blockIdx.x * ldc, len, v, size);
    if (ss == INFINITY && size < 0x7f800000u) {        // the same for the whole block, and rare: the sum again, times 2^-160; eps is nothing beside it
        const float factor = 0x1p-40f / sqrtf(block_sum_again(low, part) / (float)len);
        if (threadIdx.x == 0) scales[blockIdx.x] = scale_of(size, factor) * 0x1p-40f;
        return;
    }
    if (threadIdx.x == 0) scales[blockIdx.x] = scale_of(size, 1.0f / sqrtf(ss / (float)len + eps));
}

constexpr int ROW_MOST = 1024 * 8 * 4;    // elements that a block holds, up to four groups of eight a thread

// Groups of eight elements a thread holds: `least`, or as many as a block of 1,024 threads needs.
static inline int row_groups(int len, int least) { return len > 16384 && least < 4 ? 4 : (len > 8192 && least < 2 ? 2 : least); }
static inline int row_threads(int len, int groups)
{
    const int t = ((len + 8 * groups - 1) / (8 * groups) + 31) / 32 * 32;
    return t < 64 ? 64 : t;
}
static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T>
static int quantize(const T* x, long long ldx, int8_t* codes, long long ldc, float* scales, int n, int len, cudaStream_t stream)
{
    const bool whole = len % 8 == 0 && aligned16(x) && ldx * (long long)sizeof(T) % 16 == 0;
    if (len > ROW_MOST) {
        spy_launch(quantize_long_kernel<T>, dim3(n), dim3(1024), 0, stream, x, ldx, codes, ldc, scales, len);
        SPY_CHECK_LAUNCH("quantize_int8 (long rows)");
        return 0;
    }
    // Few rows: the row spread as wide as it goes.  Many: more groups a thread, as what a warp does once a row (reduction, barrier, division) is bought
    // once for more elements.  us with 1 / 2 / 4 / 8 groups, whole rows of bfloat16: 64 x 4,096 2.0 / 2.0 / 2.2 / 2.8, 2,048 x 4,096 7.8 / 6.6 / 7.0 / 8.0,
    // 2,048 x 12,288 - / 19.6 / 16.7 / 16.6, 24,576 x 4,096 76.3 / 58.9 / 52.9 / 51.5 (0.90 of the copy rate); of float32 64 x 4,096 1.9 / 1.9 / 2.1, 2,048 x 4,096
    // 8.4 / 7.5 / 7.8 (0.82), 24,576 x 4,096 81.1 / 73.2 / 71.8.  Others, 1 / 2 / 4 groups: float32 1,531 x 4,999 11.4 / 9.8 / 10.5, 64 x 4,999 2.2 / 2.4 / 3.1;
    // bfloat16 1,531 x 4,999 10.4 / 10.6 / 11.8.
    const bool packed = whole && sizeof(T) == 2;
    const int groups = row_groups(len, n < 1024 ? 1 : (!whole ? 2 : (packed && (long long)n * len >= (1 << 24) ? 8 : 4))), threads = row_threads(len, groups);
    if constexpr (sizeof(T) == 2) {
        if (whole) {
            auto kernel = groups == 8 ? quantize_packed_kernel<8> : groups == 4 ? quantize_packed_kernel<4> : groups == 2 ? quantize_packed_kernel<2> : quantize_packed_kernel<1>;
            spy_launch(kernel, dim3(n), dim3(threads), 0, stream, x, ldx, codes, ldc, scales, len);
            SPY_CHECK_LAUNCH("quantize_int8 (bfloat16)");
            return 0;
        }
    }
    auto kernel = whole ? (groups == 4 ? quantize_kernel<T, true, 4> : groups == 2 ? quantize_kernel<T, true, 2> : quantize_kernel<T, true, 1>)
                        : (groups == 4 ? quantize_kernel<T, false, 4> : groups == 2 ? quantize_kernel<T, false, 2> : quantize_kernel<T, false, 1>);
    spy_launch(kernel, dim3(n), dim3(threads), 0, stream, x, ldx, codes, ldc, scales, len);
    SPY_CHECK_LAUNCH("quantize_int8");
    return 0;
}

template <typename TX, typename TD, typename TW>
static int norm(TX* x, const TD* delta, int splits, long long split_stride, const int* rows, const TW* w, int8_t* codes, long long ldc, float* scales,
                int total, int n, int len, float eps, int write_back, int settled, int* status, cudaStream_t stream)
{
    const bool whole = len % 8 == 0 && aligned16(x) && aligned16(delta) && aligned16(w) && split_stride * (long long)sizeof(TD) % 16 == 0;
    // us with 1 / 2 / 4 groups a thread.  Whole rows: 64 x 5,120 2.9 / 3.7 / 3.6, 512 x 4,096 5.7 / 6.3 / 9.3, 4,096 x 5,120 37.3 / 39.3 / 40.8 (a norm with a
    // bfloat16 result 41.8).  Others: 64 x 4,999 3.5 / 4.8 / 26.1, 1,000 x 4,999 25.1 / 18.5 / 58.9; their scales' last bits follow the groups' order of summation.
    const int groups = row_groups(len, whole || n < 512 ? 1 : 2);
    auto kernel = whole ? (groups == 4 ? rmsnorm_int8_kernel<TX, TD, TW, true, 4> : groups == 2 ? rmsnorm_int8_kernel<TX, TD, TW, true, 2> : rmsnorm_int8_kernel<TX, TD, TW, true, 1>)
                        : (groups == 4 ? rmsnorm_int8_kernel<TX, TD, TW, false, 4> : groups == 2 ? rmsnorm_int8_kernel<TX, TD, TW, false, 2> : rmsnorm_int8_kernel<TX, TD, TW, false, 1>);
    spy_launch(kernel, dim3(n), dim3(row_threads(len, groups)), 0, stream, x, delta, splits, split_stride, rows, w, codes, ldc, scales, total, len, eps,
               write_back, settled, status);
    SPY_CHECK_LAUNCH("rmsnorm_int8");
    return 0;
}

static int check_codes(const char* what, const void* codes, long long ldc, int len)
{
    if (len <= 0) SPY_FAIL("%s: row length %d must be positive", what, len);
    if (!aligned16(codes) || ldc % 16 != 0) SPY_FAIL("%s: rows of codes must start on 16-byte borders (row distance %lld)", what, ldc);
    return 0;
}

}  // namespace

// x: [n, len] of dtype, rows ldx elements apart; codes: [n, len], rows ldc bytes apart (a multiple of 16); scales: [n].
extern "C" int spy_quantize_int8(const void* x, int dtype, long long ldx, int8_t* codes, long long ldc, float* scales, int n, int len, cudaStream_t stream)
{
    if (n <= 0) return 0;
    if (int rc = check_codes("quantize_int8", codes, ldc, len)) return rc;
    SPY_DISPATCH_DTYPE(dtype, T, { return quantize<T>((const T*)x, ldx, codes, ldc, scales, n, len, stream); })
    return 0;
}

// x: [total, len] of x_dtype; delta: null or `splits` stacked [*, len] arrays of delta_dtype, split_stride elements apart, added to x in order;
// rows: null or n row indices (gather), one outside x gives a row that is not a number and is reported in status (null, or two ints);
// w: [len] of w_dtype (settled: no kernel that may still run writes it); codes and scales as above.  write_back stores the sum into x and needs
// rows == null.
extern "C" int spy_rmsnorm_int8(void* x, int x_dtype, const void* delta, int delta_dtype, int splits, long long split_stride, const int* rows,
                                const void* w, int w_dtype, int8_t* codes, long long ldc, float* scales, int total, int n, int len, float eps,
                                int write_back, int settled, int* status, cudaStream_t stream)
{
    if (n <= 0) return 0;
    if (int rc = check_codes("rmsnorm_int8", codes, ldc, len)) return rc;
    if (len > ROW_MOST) SPY_FAIL("rmsnorm_int8: a row of %d elements is longer than %d", len, ROW_MOST);
    if (write_back && rows) SPY_FAIL("rmsnorm_int8: write_back with a row gather is not defined");
    if (delta && splits <= 0) SPY_FAIL("rmsnorm_int8: splits %d must be positive", splits);
    if (!delta) { delta_dtype = x_dtype; splits = 0; split_stride = 0; write_back = 0; }
    SPY_DISPATCH_DTYPE(x_dtype, TX, {
        SPY_DISPATCH_DTYPE(delta_dtype, TD, {
            SPY_DISPATCH_DTYPE(w_dtype, TW, {
                return norm<TX, TD, TW>((TX*)x, (const TD*)delta, splits, split_stride, rows, (const TW*)w, codes, ldc, scales, total, n, len, eps, write_back, settled, status, stream);
            })
        })
    })
    return 0;
}
