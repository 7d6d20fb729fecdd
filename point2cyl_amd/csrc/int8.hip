// int8.hip -- linear layers in 8-bit integers (gfx950 only): rows (points, tokens) and output channels carry one 32-bit scale each.
//
//   quantize:  s = max |row| * (1 / 127) in 32 bits, q = x / s rounded to the nearest whole number, ties to even.
//   linear:    y[r][n] = act( (sum_k q_x[r][k] q_w[n][k]) s_x[r] s_w[n] + bias[n] + add[r][n] )
// The sum is exact (32-bit integers on v_mfma_i32_32x32x32_i8, K <= 131072), the rest is 32-bit arithmetic, rounded once to the output type.
// A row with an infinite or NaN element has scale NaN and quotients 0: its outputs are NaN, other rows are not touched.  A row whose largest
// magnitude is below 2^-119 (its scale would leave the normal range) is a row of zeros, scale 0.
#include "tile_dma.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

enum { Q_F32 = 0, Q_BF16 = 1, Q_F16 = 2 };

__device__ __forceinline__ float q_get(const void *p, long long i, int dt)
{
    if (dt == Q_F32) return reinterpret_cast<const float *>(p)[i];
    if (dt == Q_BF16) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(p)[i] << 16);
    return (float)reinterpret_cast<const _Float16 *>(p)[i];
}

// scale of a row from the largest bit pattern of |x| (patterns order like the numbers, infinities and NaN on top), and the factor for the first guess
__device__ __forceinline__ float q_scale(uint32_t top, float &inv)
{
    if (top >= 0x7F800000u) { inv = 0.f; return __uint_as_float(0x7FC00000u); }
    if (top < 0x04000000u) { inv = 0.f; return 0.f; }                    // < 2^-119
    const float s = __uint_as_float(top) * (1.0f / 127.0f);
    inv = 1.0f / s;
    return s;
}

// the whole number nearest to the EXACT quotient x / s.  The guess is off by at most one, and only next to a half; x - q s fits 24 bits, so the
// fused remainder is exact and its comparison with s / 2 decides.
__device__ __forceinline__ int q_round(float x, float s, float inv)
{
    float q = rintf(x * inv);
    const float r = __builtin_fmaf(-q, s, x), a2 = 2.0f * fabsf(r), up = r < 0.f ? -1.f : 1.f;
    const bool odd = ((int)q & 1) != 0;
    if (a2 > s || (a2 == s && odd)) q += up;
    return inv == 0.f ? 0 : (int)q;
}

__device__ __forceinline__ uint32_t q_wave_max(uint32_t v) { return (uint32_t)p2c_wave_max_i32((int)v); }      // patterns of |x|: never negative

// ---- rows of up to 64 * 4 * U elements in the registers of one wave; four rows per workgroup.  VEC: 16-byte (8-byte for 16-bit types) loads
template <int DT, int U, bool VEC>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void *__restrict__ x, long long ldx, int M, int K, int Kp, int8_t *__restrict__ q,
                                                            float *__restrict__ scale)
{
    const int lane = threadIdx.x & 63;
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= M) return;
    const long long base = row * ldx;
    float v[U][4];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k = (u * 64 + lane) * 4;
        if (VEC) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] = 0.f;
            if (k < K) {
                if (DT == Q_F32) {
                    const f32x4 t = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(x) + base + k);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][e] = t[e];
                } else {
                    const uint2 t = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(x) + base + k);
                    const uint16_t w[4] = {(uint16_t)t.x, (uint16_t)(t.x >> 16), (uint16_t)t.y, (uint16_t)(t.y >> 16)};
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][e] = q_get(w, e, DT);
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] = k + e < K ? q_get(x, base + k + e, DT) : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[u][e]) & 0x7FFFFFFFu);
    }
    float inv;
    const float s = q_scale(q_wave_max(top), inv);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k = (u * 64 + lane) * 4;
        if (k < Kp) {                                          // the columns behind K hold zeros
            uint32_t o = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) o |= (uint32_t)(q_round(v[u][e], s, inv) & 0xFF) << (8 * e);
            *reinterpret_cast<uint32_t *>(q + row * Kp + k) = o;
        }
    }
    if (lane == 0) scale[row] = s;
}

// ---- longer rows: one workgroup per row, read twice (the second time out of the cache)
template <int DT>
__global__ void __launch_bounds__(256) quantize_long_kernel(const void *__restrict__ x, long long ldx, int K, int Kp, int8_t *__restrict__ q,
                                                            float *__restrict__ scale)
{
    __shared__ uint32_t red[4];
    const long long row = blockIdx.x, base = row * ldx;
    uint32_t top = 0;
    for (int k = threadIdx.x; k < K; k += 256) top = max(top, __float_as_uint(q_get(x, base + k, DT)) & 0x7FFFFFFFu);
    top = q_wave_max(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    float inv;
    const float s = q_scale(max(max(red[0], red[1]), max(red[2], red[3])), inv);
    for (int k = threadIdx.x * 4; k < Kp; k += 1024) {
        uint32_t o = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) o |= (uint32_t)(q_round(k + e < K ? q_get(x, base + k + e, DT) : 0.f, s, inv) & 0xFF) << (8 * e);
        *reinterpret_cast<uint32_t *>(q + row * Kp + k) = o;
    }
    if (threadIdx.x == 0) scale[row] = s;
}

// ---- back to floats
template <int DT>
__global__ void __launch_bounds__(256) dequantize_kernel(const int8_t *__restrict__ q, const float *__restrict__ scale, long long M, int K, int Kp,
                                                         void *__restrict__ out)
{
    const long long n = M * K;
    for (long long e = blockIdx.x * 256ll + threadIdx.x; e < n; e += gridDim.x * 256ll) {
        const long long r = e / K;
        const float v = (float)q[r * Kp + (e - r * K)] * scale[r];
        if (DT == Q_F32) reinterpret_cast<float *>(out)[e] = v;
        else if (DT == Q_BF16) reinterpret_cast<__bf16 *>(out)[e] = (__bf16)v;
        else reinterpret_cast<_Float16 *>(out)[e] = (_Float16)v;
    }
}

struct I8Epi {
    const float *sx, *sw, *bias, *add;      // bias, add may be NULL
    long long ldadd;
    void *out;
    long long ldo;
    int dtype, act, vec;                    // act: 0 none, 1 ReLU, 2 softplus; vec: 16-byte stores are aligned
    float beta, thr;
    float *so;                              // scale of the output rows (requantising kernel)
};

__device__ __forceinline__ float i8_act(float y, int act, float beta, float inv_beta, float thr)
{
    if (act == 1) return y < 0.f ? 0.f : y;                             // (NaN stays)
    if (act == 2) {
        const float bz = y * beta, e = __expf(-fabsf(bz));
        const float l1p = e < 0.0078125f ? e * (1.f - e * (0.5f - e * 0.33333334f)) : __logf(1.f + e);      // as softplus.hip
        const float v = (fmaxf(bz, 0.f) + l1p) * inv_beta;
        return bz > thr ? y : v;
    }
    return y;
}

// ---- the product.  Tile BM x BN, WR x WC waves, k-tiles of 64 bytes in NST LDS stages filled by direct copies.  The operands are handed to the
// matrix instruction weights first: a lane then holds ONE row of x and 4 consecutive output channels at a time, so the channel scales are
// registers, the row scale is one number, and a row's maximum is an in-lane affair.
template <int BM, int BN, int WR, int WC, int NST>
struct I8Tile {
    static constexpr int RB = 64, NW = WR * WC, STAGE = (BM + BN) * RB, TM = BM / WR / 32, TN = BN / WC / 32, LPW = STAGE / 1024 / NW;

    static __device__ __forceinline__ void run(const int8_t *x, long long ldx, int lastx, const int8_t *w, long long ldw, int lastw, int KT, char *smem,
                                               int wave, int lane, i32x16 (&acc)[TN][TM])
    {
        const int il = lane & 31, h = lane >> 5;
#pragma unroll
        for (int p = 0; p < TN; ++p)
#pragma unroll
            for (int q = 0; q < TM; ++q)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[p][q][r] = 0;
        auto copy = [&](int kt) {
            const int k = min(kt, KT - 1);
            char *st = smem + (kt % NST) * STAGE;
            p2c_tile_copy<BM, RB, NW>((const char *)x + (long long)k * RB, ldx, lastx, st, wave, lane);
            p2c_tile_copy<BN, RB, NW>((const char *)w + (long long)k * RB, ldw, lastw, st + BM * RB, wave, lane);
        };
#pragma unroll
        for (int s = 0; s < NST - 1; ++s) copy(s);
        const int wr = wave / WC * (BM / WR), wc = wave % WC * (BN / WC);
        for (int kt = 0; kt < KT; ++kt) {
            p2c_tile_wait<(NST - 2) * LPW>();
            copy(kt + NST - 1);
            const char *xs = smem + (kt % NST) * STAGE, *ws = xs + BM * RB;
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                i32x4 fx[TM], fw[TN];
#pragma unroll
                for (int q = 0; q < TM; ++q) fx[q] = *reinterpret_cast<const i32x4 *>(xs + p2c_tile_at<RB>(wr + q * 32 + il, 2 * s + h));
#pragma unroll
                for (int p = 0; p < TN; ++p) fw[p] = *reinterpret_cast<const i32x4 *>(ws + p2c_tile_at<RB>(wc + p * 32 + il, 2 * s + h));
#pragma unroll
                for (int p = 0; p < TN; ++p)
#pragma unroll
                    for (int q = 0; q < TM; ++q) acc[p][q] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fw[p], fx[q], acc[p][q], 0, 0, 0);
            }
        }
        p2c_tile_wait<0>();
    }
};

template <int BM, int BN, int WR, int WC, int NST>
__global__ void __launch_bounds__(64 * WR * WC) int8_linear_kernel(const int8_t *__restrict__ x, long long ldx, const int8_t *__restrict__ w, int Kp, int M,
                                                                   int N, I8Epi e, int nbn)
{
    typedef I8Tile<BM, BN, WR, WC, NST> T;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), il = lane & 31, h = lane >> 5;
    const int bm = blockIdx.x / nbn, bn = blockIdx.x - bm * nbn, m0 = bm * BM, n0 = bn * BN;
    i32x16 acc[T::TN][T::TM];
    T::run(x + (long long)m0 * ldx, ldx, M - 1 - m0, w + (long long)n0 * Kp, Kp, BN - 1, Kp / 64, smem, wave, lane, acc);

    const float inv_beta = e.act == 2 ? 1.0f / e.beta : 0.f;
    float *stage = reinterpret_cast<float *>(smem) + wave * (32 * 36);       // 32 rows x 32 channels of this wave
    const int wr = wave / WC * (BM / WR), wc = wave % WC * (BN / WC);
#pragma unroll
    for (int p = 0; p < T::TN; ++p) {
        const int c0 = n0 + wc + p * 32;
        float sw[16], bi[16];
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int k = 0; k < 4; ++k) {                                    // scales and biases are padded to the tile
                sw[4 * g + k] = e.sw[c0 + 8 * g + 4 * h + k];
                bi[4 * g + k] = e.bias ? e.bias[c0 + 8 * g + 4 * h + k] : 0.f;
            }
#pragma unroll
        for (int q = 0; q < T::TM; ++q) {
            const int r0 = m0 + wr + q * 32;
            const float sx = e.sx[min(r0 + il, M - 1)];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                f32x4 v;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] = __builtin_fmaf((float)acc[p][q][4 * g + k] * sx, sw[4 * g + k], bi[4 * g + k]);
                *reinterpret_cast<f32x4 *>(stage + il * 36 + 8 * g + 4 * h) = v;
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int t = 0; t < 2; ++t) {                                    // 8 channels of a row per lane
                const int u = lane + 64 * t, r = u >> 2, c8 = (u & 3) * 8, row = r0 + r, col = c0 + c8;
                float v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = stage[r * 36 + c8 + k];
                if (row < M && col < N) {
                    if (e.add) {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            if (col + k < N) v[k] += e.add[(long long)row * e.ldadd + col + k];
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = i8_act(v[k], e.act, e.beta, inv_beta, e.thr);
                    const long long at = (long long)row * e.ldo + col;
                    if (e.dtype == Q_F32) {
                        float *o = reinterpret_cast<float *>(e.out) + at;
                        if (e.vec && col + 8 <= N) {
                            reinterpret_cast<f32x4 *>(o)[0] = f32x4{v[0], v[1], v[2], v[3]};
                            reinterpret_cast<f32x4 *>(o)[1] = f32x4{v[4], v[5], v[6], v[7]};
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (col + k < N) o[k] = v[k];
                        }
                    } else {
                        uint16_t b[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            b[k] = e.dtype == Q_BF16 ? __builtin_bit_cast(uint16_t, (__bf16)v[k]) : __builtin_bit_cast(uint16_t, (_Float16)v[k]);
                        uint16_t *o = reinterpret_cast<uint16_t *>(e.out) + at;
                        if (e.vec && col + 8 <= N) {
                            *reinterpret_cast<u32x4 *>(o) = u32x4{b[0] | (uint32_t)b[1] << 16, b[2] | (uint32_t)b[3] << 16, b[4] | (uint32_t)b[5] << 16,
                                                                  b[6] | (uint32_t)b[7] << 16};
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                if (col + k < N) o[k] = b[k];
                        }
                    }
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
}

// ---- the product with 8-bit rows as its result: a workgroup holds whole rows (N <= BN), so their scale is known before anything is stored and the
// 32-bit activations never leave the registers.  out [M][Kp_out] int8, columns behind N zero; so [M].
template <int BM, int BN, int WR, int WC, int NST>
__global__ void __launch_bounds__(64 * WR * WC) __attribute__((amdgpu_waves_per_eu(2, 2)))
int8_requant_kernel(const int8_t *__restrict__ x, long long ldx, const int8_t *__restrict__ w, int Kp, int M, int N, I8Epi e)
{
    typedef I8Tile<BM, BN, WR, WC, NST> T;
    constexpr int LDQ = BN + 16;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), il = lane & 31, h = lane >> 5;
    const int m0 = blockIdx.x * BM;
    i32x16 acc[T::TN][T::TM];
    T::run(x + (long long)m0 * ldx, ldx, M - 1 - m0, w, Kp, BN - 1, Kp / 64, smem, wave, lane, acc);

    int8_t *qt = reinterpret_cast<int8_t *>(smem);                           // [BM][LDQ]
    uint32_t *rowtop = reinterpret_cast<uint32_t *>(smem + BM * LDQ);        // [WC][BM]
    const float inv_beta = e.act == 2 ? 1.0f / e.beta : 0.f;
    const int wr = wave / WC * (BM / WR), wc = wave % WC * (BN / WC);
    uint32_t top[T::TM];
    float sx[T::TM];
#pragma unroll
    for (int q = 0; q < T::TM; ++q) {
        top[q] = 0;
        sx[q] = e.sx[min(m0 + wr + q * 32 + il, M - 1)];
    }
#pragma unroll
    for (int p = 0; p < T::TN; ++p)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = wc + p * 32 + 8 * g + 4 * h;
            const f32x4 sw = *reinterpret_cast<const f32x4 *>(e.sw + c);
            f32x4 bi = {0.f, 0.f, 0.f, 0.f};
            if (e.bias) bi = *reinterpret_cast<const f32x4 *>(e.bias + c);
#pragma unroll
            for (int q = 0; q < T::TM; ++q)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    float v = __builtin_fmaf((float)acc[p][q][4 * g + k] * sx[q], sw[k], bi[k]);
                    if (e.add && c + k < N) v += e.add[(long long)min(m0 + wr + q * 32 + il, M - 1) * e.ldadd + c + k];
                    v = c + k < N ? i8_act(v, e.act, e.beta, inv_beta, e.thr) : 0.f;
                    top[q] = max(top[q], __float_as_uint(v) & 0x7FFFFFFFu);
                    acc[p][q][4 * g + k] = __float_as_int(v);
                }
        }
#pragma unroll
    for (int q = 0; q < T::TM; ++q) {
        const uint32_t other = (uint32_t)__shfl_xor((int)top[q], 32);
        top[q] = max(top[q], other);
        if (h == 0) rowtop[wave % WC * BM + wr + q * 32 + il] = top[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < T::TM; ++q) {
        const int r = wr + q * 32 + il;
        uint32_t t = 0;
#pragma unroll
        for (int c = 0; c < WC; ++c) t = max(t, rowtop[c * BM + r]);
        float inv;
        const float s = q_scale(t, inv);
        if (h == 0 && wave % WC == 0 && m0 + r < M) e.so[m0 + r] = s;
#pragma unroll
        for (int p = 0; p < T::TN; ++p)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uint32_t o = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) o |= (uint32_t)(q_round(__int_as_float(acc[p][q][4 * g + k]), s, inv) & 0xFF) << (8 * k);
                *reinterpret_cast<uint32_t *>(qt + r * LDQ + wc + p * 32 + 8 * g + 4 * h) = o;
            }
    }
    __syncthreads();
    const int per = (int)e.ldo / 16;                                         // 16-byte pieces of an output row
    for (int u = tid; u < BM * per; u += 64 * WR * WC) {
        const int r = u / per, c = (u - r * per) * 16;
        if (m0 + r < M) *reinterpret_cast<u32x4 *>(reinterpret_cast<int8_t *>(e.out) + (long long)(m0 + r) * e.ldo + c) = *reinterpret_cast<const u32x4 *>(qt + r * LDQ + c);
    }
}

// ---- few rows (M <= 32), rows as floats: one launch.  A workgroup owns 32 output channels; it quantises all rows into LDS (they are few and short) and its
// four waves share the k range; weights come straight from memory.
template <int DT>
__global__ void __launch_bounds__(256) int8_few_kernel(const void *__restrict__ x, long long ldx, const int8_t *__restrict__ w, int K, int Kp, int M, int N,
                                                       I8Epi e)
{
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int ldq = Kp + 16;
    int8_t *qt = reinterpret_cast<int8_t *>(smem);                           // [32][Kp + 16]
    float *sxs = reinterpret_cast<float *>(smem + 32 * ldq);                 // [32]
    int *part = reinterpret_cast<int *>(sxs + 32);                           // [3][64][17]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), il = lane & 31, h = lane >> 5, n0 = blockIdx.x * 32;
    for (int r = wave; r < M; r += 4) {
        const long long base = (long long)r * ldx;
        uint32_t top = 0;
        for (int k = lane; k < K; k += 64) top = max(top, __float_as_uint(q_get(x, base + k, DT)) & 0x7FFFFFFFu);
        float inv;
        const float s = q_scale(q_wave_max(top), inv);
        for (int k = lane * 4; k < Kp; k += 256) {
            uint32_t o = 0;
#pragma unroll
            for (int c = 0; c < 4; ++c) o |= (uint32_t)(q_round(k + c < K ? q_get(x, base + k + c, DT) : 0.f, s, inv) & 0xFF) << (8 * c);
            *reinterpret_cast<uint32_t *>(qt + r * ldq + k) = o;
        }
        if (lane == 0) sxs[r] = s;
    }
    __syncthreads();
    i32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0;
    const int8_t *wr = w + (long long)(n0 + il) * Kp + 16 * h;
    const int8_t *xr = qt + min(il, M - 1) * ldq + 16 * h;
    for (int k = wave * 32; k < Kp; k += 128)
        acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(*reinterpret_cast<const i32x4 *>(wr + k), *reinterpret_cast<const i32x4 *>(xr + k), acc, 0, 0, 0);
    if (wave) {
#pragma unroll
        for (int r = 0; r < 16; ++r) part[((wave - 1) * 64 + lane) * 17 + r] = acc[r];
    }
    __syncthreads();
    if (wave == 0 && il < M) {
        const float inv_beta = e.act == 2 ? 1.0f / e.beta : 0.f, sx = sxs[il];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int c = n0 + 8 * (r >> 2) + 4 * h + (r & 3);
            const int sum = acc[r] + part[lane * 17 + r] + part[(64 + lane) * 17 + r] + part[(128 + lane) * 17 + r];
            if (c < N) {
                float v = __builtin_fmaf((float)sum * sx, e.sw[c], e.bias ? e.bias[c] : 0.f);
                if (e.add) v += e.add[(long long)il * e.ldadd + c];
                v = i8_act(v, e.act, e.beta, inv_beta, e.thr);
                const long long at = (long long)il * e.ldo + c;
                if (e.dtype == Q_F32) reinterpret_cast<float *>(e.out)[at] = v;
                else if (e.dtype == Q_BF16) reinterpret_cast<__bf16 *>(e.out)[at] = (__bf16)v;
                else reinterpret_cast<_Float16 *>(e.out)[at] = (_Float16)v;
            }
        }
    }
}

template <int DT, bool VEC>
int quantize_launch(const void *x, long long ldx, int M, int K, int Kp, int8_t *q, float *scale, hipStream_t st)
{
    const int grid = p2c_cdiv(M, 4);
    if (Kp <= 256) hipLaunchKernelGGL((quantize_rows_kernel<DT, 1, VEC>), dim3(grid), dim3(256), 0, st, x, ldx, M, K, Kp, q, scale);
    else if (Kp <= 512) hipLaunchKernelGGL((quantize_rows_kernel<DT, 2, VEC>), dim3(grid), dim3(256), 0, st, x, ldx, M, K, Kp, q, scale);
    else if (Kp <= 1024) hipLaunchKernelGGL((quantize_rows_kernel<DT, 4, VEC>), dim3(grid), dim3(256), 0, st, x, ldx, M, K, Kp, q, scale);
    else if (Kp <= 4096) hipLaunchKernelGGL((quantize_rows_kernel<DT, 16, VEC>), dim3(grid), dim3(256), 0, st, x, ldx, M, K, Kp, q, scale);
    else hipLaunchKernelGGL((quantize_long_kernel<DT>), dim3(M), dim3(256), 0, st, x, ldx, K, Kp, q, scale);
    P2C_LAUNCH_CHECK();
    return P2C_OK;
}

template <int BM, int BN, int WR, int WC, int NST>
int linear_launch(const int8_t *x, long long ldx, const int8_t *w, int Kp, int M, int N, const I8Epi &e, hipStream_t st)
{
    typedef I8Tile<BM, BN, WR, WC, NST> T;
    constexpr int OUT = WR * WC * 32 * 36 * 4, LDS = NST * T::STAGE > OUT ? NST * T::STAGE : OUT;
    static_assert(LDS <= 160 * 1024, "");
    if (LDS > 65536) {
        const hipError_t rc = hipFuncSetAttribute((const void *)int8_linear_kernel<BM, BN, WR, WC, NST>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (rc != hipSuccess) return (int)rc;
    }
    const int nbn = p2c_cdiv(N, BN);
    hipLaunchKernelGGL((int8_linear_kernel<BM, BN, WR, WC, NST>), dim3(p2c_cdiv(M, BM) * nbn), dim3(64 * WR * WC), LDS, st, x, ldx, w, Kp, M, N, e, nbn);
    P2C_LAUNCH_CHECK();
    return P2C_OK;
}

template <int BM, int BN, int WR, int WC, int NST>
int requant_launch(const int8_t *x, long long ldx, const int8_t *w, int Kp, int M, int N, const I8Epi &e, hipStream_t st)
{
    typedef I8Tile<BM, BN, WR, WC, NST> T;
    constexpr int OUT = BM * (BN + 16) + WC * BM * 4, LDS = NST * T::STAGE > OUT ? NST * T::STAGE : OUT;
    static_assert(LDS <= 160 * 1024, "");
    if (LDS > 65536) {
        const hipError_t rc = hipFuncSetAttribute((const void *)int8_requant_kernel<BM, BN, WR, WC, NST>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (rc != hipSuccess) return (int)rc;
    }
    hipLaunchKernelGGL((int8_requant_kernel<BM, BN, WR, WC, NST>), dim3(p2c_cdiv(M, BM)), dim3(64 * WR * WC), LDS, st, x, ldx, w, Kp, M, N, e);
    P2C_LAUNCH_CHECK();
    return P2C_OK;
}

bool i8_shape_bad(long long M, int K, int Kp) { return M < 0 || M > (1ll << 30) || K < 1 || K > 131072 || Kp < K || Kp % 64; }

}  // namespace

extern "C" int p2c_int8_padded(int K) { return K < 1 ? 0 : (K + 63) / 64 * 64; }
extern "C" int p2c_int8_padded_out(int N) { return N < 1 ? 0 : (N + 255) / 256 * 256; }
extern "C" int p2c_int8_few_supported(int M, int K) { return M >= 1 && M <= 32 && K >= 1 && K <= 2048; }
extern "C" int p2c_int8_requant_supported(int N) { return N >= 1 && N <= 512; }

extern "C" int p2c_quantize_rows(const void *x, int dtype, long long ldx, int M, int K, int Kp, int8_t *q, float *scale, void *stream)
{
    if (i8_shape_bad(M, K, Kp) || dtype < 0 || dtype > 2 || ldx < 0) return P2C_EINVAL;
    if (M == 0) return P2C_OK;
    if (!x || !q || !scale) return P2C_EINVAL;
    if ((uintptr_t)q & 15) return P2C_EALIGN;
    const hipStream_t st = (hipStream_t)stream;
    const bool vec = K % 4 == 0 && ldx % 4 == 0 && ((uintptr_t)x & (dtype == 0 ? 15 : 7)) == 0;
    if (dtype == 0) return vec ? quantize_launch<Q_F32, true>(x, ldx, M, K, Kp, q, scale, st) : quantize_launch<Q_F32, false>(x, ldx, M, K, Kp, q, scale, st);
    if (dtype == 1) return vec ? quantize_launch<Q_BF16, true>(x, ldx, M, K, Kp, q, scale, st) : quantize_launch<Q_BF16, false>(x, ldx, M, K, Kp, q, scale, st);
    return vec ? quantize_launch<Q_F16, true>(x, ldx, M, K, Kp, q, scale, st) : quantize_launch<Q_F16, false>(x, ldx, M, K, Kp, q, scale, st);
}

extern "C" int p2c_dequantize_rows(const int8_t *q, const float *scale, int M, int K, int Kp, void *out, int dtype, void *stream)
{
    if (i8_shape_bad(M, K, Kp) || dtype < 0 || dtype > 2) return P2C_EINVAL;
    if (M == 0) return P2C_OK;
    if (!q || !scale || !out) return P2C_EINVAL;
    const long long n = (long long)M * K;
    const int grid = (int)((n + 1023) / 1024 < 16384 ? (n + 1023) / 1024 : 16384);
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == 0) hipLaunchKernelGGL((dequantize_kernel<Q_F32>), dim3(grid), dim3(256), 0, st, q, scale, (long long)M, K, Kp, out);
    else if (dtype == 1) hipLaunchKernelGGL((dequantize_kernel<Q_BF16>), dim3(grid), dim3(256), 0, st, q, scale, (long long)M, K, Kp, out);
    else hipLaunchKernelGGL((dequantize_kernel<Q_F16>), dim3(grid), dim3(256), 0, st, q, scale, (long long)M, K, Kp, out);
    P2C_LAUNCH_CHECK();
    return P2C_OK;
}

static int i8_epilogue(I8Epi &e, const float *sx, const float *sw, const float *bias, const float *add, long long ldadd, int act, float beta, float thr,
                       void *out, long long ldo, int dtype, int N)
{
    if (act < 0 || act > 2 || (act == 2 && !(beta > 0.f)) || dtype < 0 || dtype > 2 || ldo < N || (add && ldadd < N)) return P2C_EINVAL;
    e.sx = sx; e.sw = sw; e.bias = bias; e.add = add; e.ldadd = ldadd; e.out = out; e.ldo = ldo; e.dtype = dtype; e.act = act; e.beta = beta; e.thr = thr;
    e.so = nullptr;
    const int per = dtype == 0 ? 4 : 8;
    e.vec = ldo % per == 0 && ((uintptr_t)out & 15) == 0;
    return P2C_OK;
}

extern "C" int p2c_int8_linear(const int8_t *xq, long long ldx, const float *sx, const int8_t *wq, const float *sw, const float *bias, const float *add,
                               long long ldadd, int act, float beta, float thr, void *out, long long ldo, int dtype, int M, int N, int K, int Kp, void *stream)
{
    if (i8_shape_bad(M, K, Kp) || N < 1 || N > (1 << 20) || ldx < Kp) return P2C_EINVAL;
    I8Epi e;
    const int rc = i8_epilogue(e, sx, sw, bias, add, ldadd, act, beta, thr, out, ldo, dtype, N);
    if (rc != P2C_OK) return rc;
    if (M == 0) return P2C_OK;
    if (!xq || !sx || !wq || !sw || !out) return P2C_EINVAL;
    if (((uintptr_t)xq & 15) || ((uintptr_t)wq & 15) || ldx % 16) return P2C_EALIGN;
    const hipStream_t st = (hipStream_t)stream;
    if ((long long)p2c_cdiv(M, 256) * p2c_cdiv(N, 256) >= 192) return linear_launch<256, 256, 2, 4, 4>(xq, ldx, wq, Kp, M, N, e, st);
    if ((long long)p2c_cdiv(M, 128) * p2c_cdiv(N, 128) >= 192) return linear_launch<128, 128, 2, 2, 4>(xq, ldx, wq, Kp, M, N, e, st);
    return linear_launch<64, 64, 2, 2, 4>(xq, ldx, wq, Kp, M, N, e, st);
}

extern "C" int p2c_int8_linear_requant(const int8_t *xq, long long ldx, const float *sx, const int8_t *wq, const float *sw, const float *bias,
                                       const float *add, long long ldadd, int act, float beta, float thr, int8_t *out, int ldo, float *so, int M, int N, int K,
                                       int Kp, void *stream)
{
    if (i8_shape_bad(M, K, Kp) || N < 1 || N > 512 || ldx < Kp || ldo != (N + 63) / 64 * 64) return P2C_EINVAL;
    I8Epi e;
    const int rc = i8_epilogue(e, sx, sw, bias, add, ldadd, act, beta, thr, out, ldo, 0, N);
    if (rc != P2C_OK) return rc;
    if (M == 0) return P2C_OK;
    if (!xq || !sx || !wq || !sw || !out || !so) return P2C_EINVAL;
    if (((uintptr_t)xq & 15) || ((uintptr_t)wq & 15) || ((uintptr_t)out & 15) || ldx % 16) return P2C_EALIGN;
    e.so = so;
    const hipStream_t st = (hipStream_t)stream;
    return N <= 256 ? requant_launch<128, 256, 2, 4, 3>(xq, ldx, wq, Kp, M, N, e, st) : requant_launch<128, 512, 2, 4, 3>(xq, ldx, wq, Kp, M, N, e, st);
}

extern "C" int p2c_int8_linear_few(const void *x, int xdtype, long long ldx, const int8_t *wq, const float *sw, const float *bias, const float *add,
                                   long long ldadd, int act, float beta, float thr, void *out, long long ldo, int dtype, int M, int N, int K, int Kp,
                                   void *stream)
{
    if (i8_shape_bad(M, K, Kp) || !p2c_int8_few_supported(M, K) || N < 1 || N > (1 << 20) || xdtype < 0 || xdtype > 2 || ldx < 0) return P2C_EINVAL;
    I8Epi e;
    const int rc = i8_epilogue(e, nullptr, sw, bias, add, ldadd, act, beta, thr, out, ldo, dtype, N);
    if (rc != P2C_OK) return rc;
    if (!x || !wq || !sw || !out) return P2C_EINVAL;
    if ((uintptr_t)wq & 15) return P2C_EALIGN;
    const int lds = 32 * (Kp + 16) + 32 * 4 + 3 * 64 * 17 * 4;
    const hipStream_t st = (hipStream_t)stream;
    const int grid = p2c_cdiv(N, 32);
#define P2C_FEW(DT_)                                                                                                                          \
    do {                                                                                                                                      \
        if (lds > 65536) {                                                                                                                    \
            const hipError_t a__ = hipFuncSetAttribute((const void *)int8_few_kernel<DT_>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);  \
            if (a__ != hipSuccess) return (int)a__;                                                                                           \
        }                                                                                                                                     \
        hipLaunchKernelGGL((int8_few_kernel<DT_>), dim3(grid), dim3(256), lds, st, x, ldx, wq, K, Kp, M, N, e);                               \
    } while (0)
    if (xdtype == 0) P2C_FEW(Q_F32);
    else if (xdtype == 1) P2C_FEW(Q_BF16);
    else P2C_FEW(Q_F16);
#undef P2C_FEW
    P2C_LAUNCH_CHECK();
    return P2C_OK;
}
