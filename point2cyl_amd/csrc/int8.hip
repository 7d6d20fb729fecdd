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
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef u16x4 u16x4_u __attribute__((aligned(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef u16x8 u16x8_u __attribute__((aligned(2)));
typedef _Float16 h16x4_u __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));

constexpr int I8_CUS = 256;              // an MI355X' compute units

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

// ... of a row held in other units (factor: back to its own)
__device__ __forceinline__ float q_scale_of(uint32_t top, float factor)
{
    if (top >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
    const float t = __uint_as_float(top) * factor;
    return t < 1.5046328e-36f ? 0.f : t * (1.0f / 127.0f);                // 2^-119
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

// 4 elements from a row, wherever it starts (the memory system takes 16- and 8-byte accesses at any element's address); zeros behind K
template <int DT>
__device__ __forceinline__ f32x4 q_get4(const void *x, long long base, int k, int K)
{
    if (k + 4 <= K) {
        if (DT == Q_F32) return *reinterpret_cast<const f32x4_u *>(reinterpret_cast<const float *>(x) + base + k);
        if (DT == Q_BF16) {
            const u16x4 t = *reinterpret_cast<const u16x4_u *>(reinterpret_cast<const uint16_t *>(x) + base + k);
            return f32x4{__uint_as_float((uint32_t)t[0] << 16), __uint_as_float((uint32_t)t[1] << 16), __uint_as_float((uint32_t)t[2] << 16),
                         __uint_as_float((uint32_t)t[3] << 16)};
        }
        return __builtin_convertvector(*reinterpret_cast<const h16x4_u *>(reinterpret_cast<const _Float16 *>(x) + base + k), f32x4);
    }
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 3; ++e)
        if (k + e < K) v[e] = q_get(x, base + k + e, DT);
    return v;
}
__device__ __forceinline__ uint32_t q_top4(f32x4 v, uint32_t top)
{
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    return top;
}
__device__ __forceinline__ uint32_t q_pack4(f32x4 v, float s, float inv)
{
    uint32_t o = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) o |= (uint32_t)(q_round(v[e], s, inv) & 0xFF) << (8 * e);
    return o;
}

// ---- rows held in registers while their maximum is found: one wave per row (four rows per workgroup) or, LONG, one workgroup per row; U pieces of 4 a lane
template <int DT, int U, bool LONG>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const void *__restrict__ x, long long ldx, int M, int K, int Kp, int8_t *__restrict__ q,
                                                            float *__restrict__ scale)
{
    __shared__ uint32_t red[4];
    constexpr int T = LONG ? 256 : 64;
    const int t = LONG ? threadIdx.x : threadIdx.x & 63;
    const long long row = LONG ? (long long)blockIdx.x : (long long)blockIdx.x * 4 + (threadIdx.x >> 6), base = row * ldx;
    if (row >= M) return;
    f32x4 v[U];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = q_get4<DT>(x, base, (u * T + t) * 4, K);
#pragma unroll
    for (int u = 0; u < U; ++u) top = q_top4(v[u], top);
    top = q_wave_max(top);
    if (LONG) {
        if ((t & 63) == 0) red[t >> 6] = top;
        __syncthreads();
        top = max(max(red[0], red[1]), max(red[2], red[3]));
    }
    float inv;
    const float s = q_scale(top, inv);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int k = (u * T + t) * 4;
        if (k < Kp) *reinterpret_cast<uint32_t *>(q + row * Kp + k) = q_pack4(v[u], s, inv);      // the columns behind K hold zeros
    }
    if (t == 0) scale[row] = s;
}

// ---- longer rows: one workgroup per row, read twice (the second time out of the cache)
template <int DT>
__global__ void __launch_bounds__(256) quantize_long_kernel(const void *__restrict__ x, long long ldx, int K, int Kp, int8_t *__restrict__ q,
                                                            float *__restrict__ scale)
{
    __shared__ uint32_t red[4];
    const long long row = blockIdx.x, base = row * ldx;
    uint32_t top = 0;
    for (int k = threadIdx.x * 4; k < Kp; k += 1024) top = q_top4(q_get4<DT>(x, base, k, K), top);
    top = q_wave_max(top);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    float inv;
    const float s = q_scale(max(max(red[0], red[1]), max(red[2], red[3])), inv);
    for (int k = threadIdx.x * 4; k < Kp; k += 1024) *reinterpret_cast<uint32_t *>(q + row * Kp + k) = q_pack4(q_get4<DT>(x, base, k, K), s, inv);
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
    int dtype, act;                         // act: 0 none, 1 ReLU, 2 softplus
    float beta, thr;
    float *so;                              // scale of the output rows (requantising kernel)
};

template <int ACT>
__device__ __forceinline__ float i8_act(float y, float beta, float inv_beta, float thr)
{
    if (ACT == 1) return y < 0.f ? 0.f : y;                             // (NaN stays)
    if (ACT == 2) {
        const float bz = y * beta, e = __expf(-fabsf(bz));
        const float l1p = e < 0.0078125f ? e * (1.f - e * (0.5f - e * 0.33333334f)) : __logf(1.f + e);      // as softplus.hip
        return bz > thr ? y : (fmaxf(bz, 0.f) + l1p) * inv_beta;
    }
    return y;
}

// log2(1 + 2^z) = max(z, 0) + log2(1 + e), e = 2^-|z|: the softplus in units where it costs one exponential and a polynomial (log2(1 + e) / e on
// [0, 1], degree 7, relative error 4e-7 - fitted by reweighted least squares).  The requantising epilogue is bound by its vector instructions.
// The coefficients are held in scalar registers (as literals they cost a move or eight bytes each time).
struct I8Poly {
    float c[8];
    __device__ __forceinline__ I8Poly()
        : c{1.4426947832107544f, -0.7213100790977478f, 0.48006361722946167f, -0.35339438915252686f, 0.2560085356235504f, -0.15535026788711548f,
            0.06360677629709244f, -0.012319165281951427f}
    {
#pragma unroll
        for (int k = 0; k < 8; ++k) asm("" : "+s"(c[k]));
    }
};
__device__ __forceinline__ float i8_softplus2(float z, const I8Poly &k)
{
    const float e = __builtin_amdgcn_exp2f(-fabsf(z));
    float p = k.c[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) p = __builtin_fmaf(p, e, k.c[i]);
    float m;
    asm("v_max_f32 %0, 0, %1" : "=v"(m) : "v"(z));                            // (fmaxf quiets its operand first: one more instruction an element)
    return __builtin_fmaf(p, e, m);
}

// ---- the product.  Tile BM x BN, WR x WC waves, k-tiles of 64 bytes in NST LDS stages filled by direct copies.  The operands are handed to the
// matrix instruction weights first: a lane then holds ONE row of x and 4 consecutive output channels at a time, so the channel scales are
// registers, the row scale is one number, and a row's maximum is an in-lane affair.
// A k-tile is multiplied in two halves; the reads of the next half and the copies of a later k-tile are issued between the products of this one, because
// instructions issue in order and a wave behind a queue of copies does not multiply.  16384 x 4096 x 4096: 299 us with copies, reads and products in turn,
// 270 so (20 calls out of idle; in a long run 236 = 2330 TOP/s, a large library product without scales, bias or rounding 2210).
template <int BM, int BN, int WR, int WC, int NST>
struct I8Tile {
    static constexpr int RB = 64, NW = WR * WC, STAGE = (BM + BN) * RB, TM = BM / WR / 32, TN = BN / WC / 32;
    static constexpr int NXC = BM * RB / 1024 / NW, NWC = BN * RB / 1024 / NW, LPW = NXC + NWC;       // copies per wave and k-tile: of x, of w, both
    static_assert(BM * RB % (1024 * NW) == 0 && BN * RB % (1024 * NW) == 0, "the same number of copies in every wave");

    // A copy's source is a scalar base plus a lane's 32-bit offset.  x: rows behind `last` are read from row `last` (their results are never stored).
    struct RowsX {
        const char *base;
        unsigned at[NXC];
        __device__ __forceinline__ void set(const int8_t *x, long long ld, int last, int wave, int lane)
        {
            base = (const char *)x;
#pragma unroll
            for (int i = 0; i < NXC; ++i) at[i] = p2c_tile_source<RB>(wave + i * NW, (int)ld, last, lane);
        }
    };
    // w: never short of a row, and a piece's 16 rows repeat the swizzle, so its pieces differ by a scalar
    struct RowsW {
        const char *base;
        unsigned at;
        long long step;
        __device__ __forceinline__ void set(const int8_t *w, int ld, int wave, int lane)
        {
            base = (const char *)w + (long long)wave * 16 * ld;
            at = p2c_tile_source<RB>(0, ld, 15, lane);
            step = (long long)NW * 16 * ld;
        }
    };

    // One tile's sums.  FLOW: a tile follows this one with sources (xn, wn), and what is copied past this tile's end are its first k-tiles: only the `first`
    // tile of a workgroup waits for memory.  KT >= NST then.  Without FLOW the stages are free afterwards.  now: the stage to begin with.
    // meanwhile(): done while the very first operands are on their way.
    template <bool FLOW, class F>
    static __device__ __forceinline__ void run(const RowsX &sx, const RowsW &sw, const RowsX &xn, const RowsW &wn, int KT, bool first, int &now, char *smem, int wave, int lane, i32x16 (&acc)[TN][TM], F meanwhile)
    {
        const int il = lane & 31, h = lane >> 5;
#pragma unroll
        for (int p = 0; p < TN; ++p)
#pragma unroll
            for (int q = 0; q < TM; ++q)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[p][q][r] = 0;
        auto copy = [&](int kt, int stage, int i) {  // (nothing follows: the last k-tile again, into a stage that is not multiplied: the count in flight stays exact)
            const bool past = FLOW && kt >= KT;
            const long long k = (long long)(past ? kt - KT : min(kt, KT - 1)) * RB;
            char *st = smem + stage * STAGE + wave * 1024;
            if (i < NXC) p2c_tile_piece((past ? xn.base : sx.base) + k + (past ? xn.at[i] : sx.at[i]), st + i * NW * 1024);
            else p2c_tile_piece((past ? wn.base : sw.base) + k + (i - NXC) * sw.step + sw.at, st + BM * RB + (i - NXC) * NW * 1024);
        };
        if (first) {
#pragma unroll
            for (int s = 0; s < NST; ++s)
#pragma unroll
                for (int i = 0; i < LPW; ++i) copy(s, s, i);
            meanwhile();
            p2c_tile_wait<(NST - 1) * LPW>();
        }
        const int wr = wave / WC * (BM / WR), wc = wave % WC * (BN / WC);
        struct Frags { i32x4 x[TM], w[TN]; };
        constexpr int R = TM + TN, M = TM * TN;
        auto read = [&](Frags &f, int stage, int half, int i) {              // fragment i of R
            const char *xs = smem + stage * STAGE, *ws = xs + BM * RB;
            if (i < TM) f.x[i] = *reinterpret_cast<const i32x4 *>(xs + p2c_tile_at<RB>(wr + i * 32 + il, 2 * half + h));
            else f.w[i - TM] = *reinterpret_cast<const i32x4 *>(ws + p2c_tile_at<RB>(wc + (i - TM) * 32 + il, 2 * half + h));
        };
        // a half's products; after each, its share of the next half's reads and of what else is to be issued
        auto multiply = [&](const Frags &f, Frags &g, int stage, int half, auto then) {
#pragma unroll
            for (int p = 0; p < TN; ++p)
#pragma unroll
                for (int q = 0; q < TM; ++q) {
                    const int n = p * TM + q;
                    acc[p][q] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.w[p], f.x[q], acc[p][q], 0, 0, 0);
#pragma unroll
                    for (int i = 2 * n; i < (n + 1 == M ? R : 2 * n + 2) && i < R; ++i) read(g, stage, half, i);
                    then(n);
                    asm volatile("" ::: "memory");
                    __builtin_amdgcn_sched_barrier(0);
                }
        };
        Frags f0, f1;
#pragma unroll
        for (int i = 0; i < R; ++i) read(f0, now, 0, i);
        for (int kt = 0; kt < KT; ++kt) {
            const int next = now + 1 == NST ? 0 : now + 1;
            __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 3 << 14);              // f0 has arrived (lgkmcnt 0): known before the next reads are issued, or the products would wait for those
            multiply(f0, f1, now, 1, [](int) {});
            // k-tile kt + 1 is here; everybody has read kt.  (At the start of a following tile the last one's stores are among what is in flight: they may
            // end out of turn, so the wait is for everything.)
            if (FLOW && !first && kt == 0) p2c_tile_wait<0>();
            else p2c_tile_wait<(NST - 2) * LPW>();
            multiply(f1, f0, next, 0, [&](int n) {
#pragma unroll
                for (int i = n * LPW / M; i < (n + 1) * LPW / M; ++i) copy(kt + NST, now, i);
            });
            now = next;
        }
        if (!FLOW) p2c_tile_wait<0>();
    }
};

// Scales and biases of BN channels (they are padded that far; `behind`: bias of channels that do not exist) for the LDS.  load() before the operands'
// copies, put() after: a load behind them could only be waited for with all of them.
template <int BN, int NT>
struct I8Factors {
    float sw[(BN + NT - 1) / NT], bi[(BN + NT - 1) / NT];
    __device__ __forceinline__ void load(const I8Epi &e, int n0, int N, int tid, float behind)
    {
#pragma unroll
        for (int c = 0; c < BN; c += NT)
            if (BN % NT == 0 || c + tid < BN) {
                sw[c / NT] = e.sw[n0 + c + tid];
                bi[c / NT] = n0 + c + tid >= N ? behind : e.bias ? e.bias[n0 + c + tid] : 0.f;
            }
    }
    __device__ __forceinline__ void put(float *f, int tid, float unit) const
    {
#pragma unroll
        for (int c = 0; c < BN; c += NT)
            if (BN % NT == 0 || c + tid < BN) {
                f[c + tid] = sw[c / NT] * unit;
                f[BN + c + tid] = bi[c / NT] * unit;
            }
    }
};

__device__ __forceinline__ void i8_store4(float *row, int c, int N, f32x4 v)
{
    if (c + 4 <= N) { *reinterpret_cast<f32x4_u *>(row + c) = v; return; }
#pragma unroll
    for (int k = 0; k < 3; ++k)
        if (c + k < N) row[c + k] = v[k];
}
__device__ __forceinline__ void i8_store8(uint16_t *row, int c, int N, u16x8 v)
{
    if (c + 8 <= N) { *reinterpret_cast<u16x8_u *>(row + c) = v; return; }
#pragma unroll
    for (int k = 0; k < 7; ++k)
        if (c + k < N) row[c + k] = v[k];
}

// LDS: operand stages; 32 rows of a wave's result in fp32, PC pieces of 32 channels wide (with FLOW one, behind the stages, which are being filled for
// the next tile); factors
template <int WAVES, int BN, int TN, int OPS, bool FLOW>
struct I8Linear {
    static constexpr int PC = FLOW ? 1 : TN, LDF = PC * 128 + 16, PIECE = 32 * LDF, OUT = WAVES * PIECE, STAGE = FLOW ? OPS : 0;
    static constexpr int FACT = FLOW ? OPS + OUT : OPS > OUT ? OPS : OUT, LDS = FACT + 2 * BN * 4;
};

template <int BM, int BN, int WR, int WC, int NST, bool FLOW, int ACT>
__global__ void __launch_bounds__(64 * WR * WC, 2) int8_linear_kernel(const int8_t *__restrict__ x, const int8_t *__restrict__ w, long long ldx, int Kp,
                                                                      int M, int N, int nbn, I8Epi e)
{
    typedef I8Tile<BM, BN, WR, WC, NST> T;
    typedef I8Linear<WR * WC, BN, T::TN, NST * T::STAGE, FLOW> L;
    static_assert(T::TN <= 2, "32 rows in 16 bits fit where one piece in 32 does");
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wr = wave / WC * (BM / WR), wc = wave % WC * (BN / WC);
    float *fact = reinterpret_cast<float *>(smem + L::FACT);
    char *stage = smem + L::STAGE + wave * L::PIECE;
    const float inv_beta = ACT == 2 ? 1.0f / e.beta : 0.f;
    const int tiles = (M + BM - 1) / BM * nbn;
    typename T::RowsX xs, xn;
    typename T::RowsW ws, wn;
    int now = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    int tid = threadIdx.x;
    if (FLOW) asm volatile("" : "+v"(tid));                                  // (the addresses made of it are made again for every tile: kept, they cost registers)
    const int lane = tid & 63, il = lane & 31, h = lane >> 5;
    const int bm = tile / nbn, bn = tile - bm * nbn, m0 = bm * BM, n0 = bn * BN, c0 = n0 + wc;
    const bool first = !FLOW || tile == (int)blockIdx.x;
    if (first) {
        xs.set(x + (long long)m0 * ldx, ldx, M - 1 - m0, wave, lane);
        ws.set(w + (long long)n0 * Kp, Kp, wave, lane);
    }
    if (FLOW) {
        const int t1 = tile + (int)gridDim.x < tiles ? tile + (int)gridDim.x : tile, bm1 = t1 / nbn;          // (behind the last tile: itself once more)
        xn.set(x + (long long)bm1 * BM * ldx, ldx, M - 1 - bm1 * BM, wave, lane);
        wn.set(w + (long long)(t1 - bm1 * nbn) * BN * Kp, Kp, wave, lane);
    } else {
        xn = xs;
        wn = ws;
    }
    float sx[T::TM];
#pragma unroll
    for (int q = 0; q < T::TM; ++q) sx[q] = e.sx[min(m0 + wr + q * 32 + il, M - 1)];
    I8Factors<BN, 64 * WR * WC> fa;
    fa.load(e, n0, N, tid, 0.f);
    i32x16 acc[T::TN][T::TM];
    T::template run<FLOW>(xs, ws, xn, wn, Kp / 64, first, now, smem, wave, lane, acc, [&]() { if (!FLOW) fa.put(fact, tid, 1.0f); });
    if (FLOW) {
        fa.put(fact, tid, 1.0f);                                             // (everybody is through with the last tile's)
        __syncthreads();
    }

    // epilogue, 32 rows of a wave at a time: finished in the registers (a lane: one row, 4 consecutive channels), through LDS in the output's type, out in
    // 16-byte pieces along the rows.  What differs between calls is decided per piece, not per element.
    constexpr int PC = L::PC, LDF = L::LDF, LDB = T::TN * 64 + 16;           // bytes of a staged row, 32- and 16-bit outputs
#pragma unroll
    for (int q = 0; q < T::TM; ++q) {
        const int r0 = m0 + wr + q * 32;
#pragma unroll
        for (int p = 0; p < T::TN; ++p) {
            f32x4 v[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int c = wc + p * 32 + 8 * g + 4 * h;
                const f32x4 sw = *reinterpret_cast<const f32x4 *>(fact + c), bi = *reinterpret_cast<const f32x4 *>(fact + BN + c);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[g][k] = __builtin_fmaf((float)acc[p][q][4 * g + k] * sx[q], sw[k], bi[k]);
            }
            if (e.add) {
#pragma unroll
                for (int g = 0; g < 4; ++g) v[g] += q_get4<Q_F32>(e.add, (long long)min(r0 + il, M - 1) * e.ldadd, c0 + p * 32 + 8 * g + 4 * h, N);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v[g][k] = i8_act<ACT>(v[g][k], e.beta, inv_beta, e.thr);
                    asm("" : "+v"(v[g][k]));                                 // one value for the three stores below, not three expressions
                }
            if (e.dtype == Q_F32) {
#pragma unroll
                for (int g = 0; g < 4; ++g) *reinterpret_cast<f32x4 *>(stage + il * LDF + (p % PC * 32 + 8 * g + 4 * h) * 4) = v[g];
                if (p % PC == PC - 1) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
                    for (int t = 0; t < 4 * PC; ++t) {                       // (stores need no more than an element's alignment)
                        const int u = lane + 64 * t, r = u / (8 * PC), c4 = u % (8 * PC) * 4;
                        if (r0 + r < M)
                            i8_store4(reinterpret_cast<float *>(e.out) + (long long)(r0 + r) * e.ldo, c0 + (p - PC + 1) * 32 + c4, N, *reinterpret_cast<const f32x4 *>(stage + r * LDF + c4 * 4));
                    }
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                }
            } else if (e.dtype == Q_BF16) {
#pragma unroll
                for (int g = 0; g < 4; ++g) *reinterpret_cast<bf16x4 *>(stage + il * LDB + (p * 32 + 8 * g + 4 * h) * 2) = __builtin_convertvector(v[g], bf16x4);
            } else {
#pragma unroll
                for (int g = 0; g < 4; ++g) *reinterpret_cast<h16x4 *>(stage + il * LDB + (p * 32 + 8 * g + 4 * h) * 2) = __builtin_convertvector(v[g], h16x4);
            }
        }
        if (e.dtype != Q_F32) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int t = 0; t < 2 * T::TN; ++t) {
                const int u = lane + 64 * t, r = u / (4 * T::TN), c8 = u % (4 * T::TN) * 8;
                if (r0 + r < M) i8_store8(reinterpret_cast<uint16_t *>(e.out) + (long long)(r0 + r) * e.ldo, c0 + c8, N, *reinterpret_cast<const u16x8 *>(stage + r * LDB + c8 * 2));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
    if (!FLOW) break;
    xs = xn;
    ws = wn;
    }
    if (FLOW) p2c_tile_wait<0>();                                            // the copies past the last tile have landed before the LDS is given back
}

// LDS of the requantising kernel: operand stages; rows of the result, maxima (with FLOW behind the stages, which are being filled for the next tile); factors
template <int BM, int BN, int WC, int OPS, bool FLOW>
struct I8Requant {
    static constexpr int LDQ = BN + 16, OUT = BM * LDQ + (WC + 1) * BM * 4, QT = FLOW ? OPS : 0, TOP = QT + BM * LDQ;
    static constexpr int FACT = FLOW ? OPS + OUT : OPS > OUT ? OPS : OUT, LDS = FACT + 2 * BN * 4;
};

// ---- the product with 8-bit rows as its result: a workgroup holds whole rows (N <= BN), so their scale is known before anything is stored and the
// 32-bit activations never leave the registers.  out [M][ldo] int8, columns behind N zero; so [M].  Softplus is computed in units of log2(e) / beta
// (scale and bias carry the factor, the row's scale divides it out).  64 rows in four waves, two workgroups per CU; with many rows 128 in eight waves, one
// workgroup per CU that goes from tile to tile (FLOW): the next tile's operands arrive during the epilogue, and the weights are read half as often.
// 262144 x 512 x 512 with softplus: 191 us and 180 in turn, from 20 calls out of idle; in a long run of calls the second takes 159.  Of the 191's clocks, by leaving out one part
// at a time, 30 % went with the copies (a tile of 64 rows reads all the weights: 1.2 GB through the L2s), 12 % with the activation (17 vector instructions per
// element and an exponential in the whole epilogue), 10 % with the stores, 4 % with the products; what the other 44 % go with is not known.
template <int BM, int BN, int WR, int WC, int NST, bool FLOW, int ACT>
__global__ void __launch_bounds__(64 * WR * WC, 2) int8_requant_kernel(const int8_t *__restrict__ x, const int8_t *__restrict__ w, long long ldx, int Kp,
                                                                       int M, int N, I8Epi e)
{
    typedef I8Tile<BM, BN, WR, WC, NST> T;
    typedef I8Requant<BM, BN, WC, NST * T::STAGE, FLOW> L;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const float unit = ACT == 2 ? e.beta * 1.44269504f : 1.0f;
    float *fact = reinterpret_cast<float *>(smem + L::FACT);
    int8_t *qt = reinterpret_cast<int8_t *>(smem + L::QT);                   // [BM][LDQ]
    float *rowtop = reinterpret_cast<float *>(smem + L::TOP);                // [WC][BM]
    uint32_t *live = reinterpret_cast<uint32_t *>(rowtop + WC * BM);         // [BM]: all ones, or zero for a row without a finite, normal scale
    constexpr int LDQ = L::LDQ;
    const int wr = wave / WC * (BM / WR), wc = wave % WC * (BN / WC);
    typename T::RowsX xs, xn;
    typename T::RowsW ws;
    const int tiles = (M + BM - 1) / BM;
    int now = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));                                            // (the addresses made of it are made again for every tile: kept, they cost 40 registers)
    const int lane = tid & 63, il = lane & 31, h = lane >> 5, m0 = tile * BM;
    ws.set(w, Kp, wave, lane);
    const bool first = !FLOW || tile == (int)blockIdx.x;
    if (first) xs.set(x + (long long)m0 * ldx, ldx, M - 1 - m0, wave, lane);
    const int m1 = tile + (int)gridDim.x < tiles ? m0 + (int)gridDim.x * BM : m0;              // (behind the last tile: itself once more)
    if (FLOW) xn.set(x + (long long)m1 * ldx, ldx, M - 1 - m1, wave, lane);
    else xn = xs;
    float top[T::TM], sx[T::TM];
#pragma unroll
    for (int q = 0; q < T::TM; ++q) {
        top[q] = 0.f;
        sx[q] = e.sx[min(m0 + wr + q * 32 + il, M - 1)];
    }
    I8Factors<BN, 64 * WR * WC> fa;
    if (first) fa.load(e, 0, N, tid, ACT == 2 ? -__builtin_inff() : 0.f);
    i32x16 acc[T::TN][T::TM];
    T::template run<FLOW>(xs, ws, xn, ws, Kp / 64, first, now, smem, wave, lane, acc, [&]() { fa.put(fact, tid, unit); });
    const I8Poly poly;
    // (softplus of the channels behind N: log2(1 + 2^-inf) = 0)
#pragma unroll
    for (int p = 0; p < T::TN; ++p) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = wc + p * 32 + 8 * g + 4 * h;
            const f32x4 sw = *reinterpret_cast<const f32x4 *>(fact + c), bi = *reinterpret_cast<const f32x4 *>(fact + BN + c);
#pragma unroll
            for (int q = 0; q < T::TM; ++q)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    acc[p][q][4 * g + k] = __float_as_int(__builtin_fmaf((float)acc[p][q][4 * g + k] * sx[q], sw[k], bi[k]));
        }
        if (e.add) {
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
                for (int q = 0; q < T::TM; ++q) {
                    const f32x4 a4 = q_get4<Q_F32>(e.add, (long long)min(m0 + wr + q * 32 + il, M - 1) * e.ldadd, wc + p * 32 + 8 * g + 4 * h, N);
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[p][q][4 * g + k] = __float_as_int(__builtin_fmaf(a4[k], unit, __int_as_float(acc[p][q][4 * g + k])));
                }
        }
#pragma unroll
        for (int q = 0; q < T::TM; ++q)
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                float v = __int_as_float(acc[p][q][k]);
                if (ACT == 1) v = v < 0.f ? 0.f : v;
                if (ACT == 2) v = i8_softplus2(v, poly);
                top[q] = __builtin_elementwise_maximum(top[q], fabsf(v));        // (a NaN wins)
                acc[p][q][k] = __float_as_int(v);
            }
    }
#pragma unroll
    for (int q = 0; q < T::TM; ++q) {
        top[q] = __builtin_elementwise_maximum(top[q], __shfl_xor(top[q], 32));
        if (h == 0) rowtop[wave % WC * BM + wr + q * 32 + il] = top[q];
    }
    __syncthreads();
    float magic = 12582912.0f;
    asm("" : "+s"(magic));
#pragma unroll
    for (int q = 0; q < T::TM; ++q) {
        const int r = wr + q * 32 + il;
        float t = 0.f;
#pragma unroll
        for (int c = 0; c < WC; ++c) t = __builtin_elementwise_maximum(t, rowtop[c * BM + r]);
        const float s = q_scale_of(__float_as_uint(t) & 0x7FFFFFFFu, 1.0f / unit);
        // v / (max / 127) rounded to the nearest: the low byte of v * inv + 1.5 2^23
        const float inv = 127.0f / t;
        if (h == 0 && wave % WC == 0) {
            live[r] = s > 0.f ? 0xFFFFFFFFu : 0u;
            if (m0 + r < M) e.so[m0 + r] = s;
        }
#pragma unroll
        for (int p = 0; p < T::TN; ++p)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uint32_t b[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(__builtin_fmaf(__int_as_float(acc[p][q][4 * g + k]), inv, magic));
                const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000C0Cu);
                *reinterpret_cast<uint32_t *>(qt + r * LDQ + wc + p * 32 + 8 * g + 4 * h) = lo | hi;
            }
    }
    __syncthreads();
    const int per = (int)e.ldo / 16;                                         // 16-byte pieces of an output row
    for (int u = tid; u < BM * per; u += 64 * WR * WC) {
        const int r = u / per, c = (u - r * per) * 16;
        if (m0 + r < M)
            *reinterpret_cast<u32x4 *>(reinterpret_cast<int8_t *>(e.out) + (long long)(m0 + r) * e.ldo + c) = *reinterpret_cast<const u32x4 *>(qt + r * LDQ + c) & live[r];
    }
    if (!FLOW) break;
    xs = xn;
    }
    if (FLOW) p2c_tile_wait<0>();                                            // the copies past the last tile have landed before the LDS is given back
}

// ---- few rows (M <= 32), rows as floats: one launch.  A workgroup owns 32 output channels; it quantises all rows into LDS (they are few and short)
// while its first weights are on their way, its four waves share the k range, weights come straight from memory.
template <int DT>
__global__ void __launch_bounds__(256) int8_few_kernel(const void *__restrict__ x, long long ldx, const int8_t *__restrict__ w, int K, int Kp, int M, int N,
                                                       I8Epi e)
{
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int ldq = Kp + 16;
    int8_t *qt = reinterpret_cast<int8_t *>(smem);                           // [32][Kp + 16]
    float *sxs = reinterpret_cast<float *>(smem + 32 * ldq);                 // [32]
    int *part = reinterpret_cast<int *>(sxs + 32);                           // [4][32 rows][36]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), il = lane & 31, h = lane >> 5, n0 = blockIdx.x * 32;
    const int8_t *wr = w + (long long)(n0 + il) * Kp + 16 * h;
    const int KS = Kp / 32;                                                  // k-steps; wave w takes w, w + 4, ...
    i32x4 ahead[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ahead[i] = *reinterpret_cast<const i32x4 *>(wr + 32 * min(wave + 4 * i, KS - 1));
    for (int r = wave; r < M; r += 4) {
        const long long base = (long long)r * ldx;
        f32x4 v[8];
        uint32_t top = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (u * 256 < Kp) v[u] = q_get4<DT>(x, base, (u * 64 + lane) * 4, K);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (u * 256 < Kp) top = q_top4(v[u], top);
        float inv;
        const float s = q_scale(q_wave_max(top), inv);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int k = (u * 64 + lane) * 4;
            if (k < Kp) *reinterpret_cast<uint32_t *>(qt + r * ldq + k) = q_pack4(v[u], s, inv);
        }
        if (lane == 0) sxs[r] = s;
    }
    __syncthreads();
    i32x16 acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] = 0;
    const int8_t *xr = qt + min(il, M - 1) * ldq + 16 * h;
    for (int k0 = wave; k0 < KS; k0 += 16) {
        i32x4 cur[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            cur[i] = ahead[i];
            ahead[i] = *reinterpret_cast<const i32x4 *>(wr + 32 * min(k0 + 16 + 4 * i, KS - 1));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (k0 + 4 * i < KS) acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(cur[i], *reinterpret_cast<const i32x4 *>(xr + 32 * (k0 + 4 * i)), acc, 0, 0, 0);
    }
#pragma unroll
    for (int g = 0; g < 4; ++g)
        *reinterpret_cast<i32x4 *>(part + (wave * 32 + il) * 36 + 8 * g + 4 * h) = i32x4{acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
    __syncthreads();
    const float inv_beta = e.act == 2 ? 1.0f / e.beta : 0.f;
    for (int u = tid; u < M * 32; u += 256) {
        const int r = u >> 5, c = u & 31, n = n0 + c;
        if (n < N) {
            const int sum = part[r * 36 + c] + part[(32 + r) * 36 + c] + part[(64 + r) * 36 + c] + part[(96 + r) * 36 + c];
            float v = __builtin_fmaf((float)sum * sxs[r], e.sw[n], e.bias ? e.bias[n] : 0.f);
            if (e.add) v += e.add[(long long)r * e.ldadd + n];
            v = e.act == 0 ? v : e.act == 1 ? i8_act<1>(v, e.beta, inv_beta, e.thr) : i8_act<2>(v, e.beta, inv_beta, e.thr);
            const long long at = (long long)r * e.ldo + n;
            if (e.dtype == Q_F32) reinterpret_cast<float *>(e.out)[at] = v;
            else if (e.dtype == Q_BF16) reinterpret_cast<__bf16 *>(e.out)[at] = (__bf16)v;
            else reinterpret_cast<_Float16 *>(e.out)[at] = (_Float16)v;
        }
    }
}

// Rows of one launch: a grid holds fewer than 2^32 threads, and a workgroup of 256 takes four rows of up to 1024 elements or one longer row.
inline int quantize_rows_at_once(int Kp) { return Kp <= 1024 ? 1 << 25 : 1 << 23; }

// A row in a wave up to 1024 elements: 262144 x 512 fp32 in 113 us = 5.9 TB/s.  Longer ones in a workgroup.
template <int DT>
int quantize_once(const void *x, long long ldx, int M, int K, int Kp, int8_t *q, float *scale, hipStream_t st)
{
    const int grid = p2c_cdiv(M, 4);
#define P2C_QUANT(U_, LONG_) \
    hipLaunchKernelGGL((quantize_rows_kernel<DT, U_, LONG_>), dim3((LONG_) ? M : grid), dim3(256), 0, st, x, ldx, M, K, Kp, q, scale)
    if (Kp <= 256) P2C_QUANT(1, false);
    else if (Kp <= 512) P2C_QUANT(2, false);
    else if (Kp <= 1024) P2C_QUANT(4, false);
    else if (Kp <= 2048) P2C_QUANT(2, true);
    else if (Kp <= 4096) P2C_QUANT(4, true);
    else hipLaunchKernelGGL((quantize_long_kernel<DT>), dim3(M), dim3(256), 0, st, x, ldx, K, Kp, q, scale);
#undef P2C_QUANT
    P2C_LAUNCH_CHECK();
    return P2C_OK;
}
template <int DT>
int quantize_launch(const void *x, long long ldx, int M, int K, int Kp, int8_t *q, float *scale, hipStream_t st)
{
    const long long width = DT == Q_F32 ? 4 : 2, most = quantize_rows_at_once(Kp);
    for (long long r = 0; r < M; r += most) {
        const int rc = quantize_once<DT>((const char *)x + r * ldx * width, ldx, (int)(M - r < most ? M - r : most), K, Kp, q + r * Kp, scale + r, st);
        if (rc != P2C_OK) return rc;
    }
    return P2C_OK;
}

template <int BM, int BN, int WR, int WC, int NST, bool FLOW, int ACT>
int linear_launch(const int8_t *x, long long ldx, const int8_t *w, int Kp, int M, int N, const I8Epi &e, hipStream_t st)
{
    typedef I8Tile<BM, BN, WR, WC, NST> T;
    constexpr int LDS = I8Linear<WR * WC, BN, T::TN, NST * T::STAGE, FLOW>::LDS;
    static_assert(LDS <= 160 * 1024, "");
    if (LDS > 65536) {
        const hipError_t rc = hipFuncSetAttribute((const void *)int8_linear_kernel<BM, BN, WR, WC, NST, FLOW, ACT>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (rc != hipSuccess) return (int)rc;
    }
    const int nbn = p2c_cdiv(N, BN), tiles = p2c_cdiv(M, BM) * nbn, grid = FLOW && tiles > I8_CUS ? I8_CUS : tiles;
    hipLaunchKernelGGL((int8_linear_kernel<BM, BN, WR, WC, NST, FLOW, ACT>), dim3(grid), dim3(64 * WR * WC), LDS, st, x, w, ldx, Kp, M, N, nbn, e);
    P2C_LAUNCH_CHECK();
    return P2C_OK;
}
template <int BM, int BN, int WR, int WC, int NST, bool FLOW>
int linear_any(const int8_t *x, long long ldx, const int8_t *w, int Kp, int M, int N, const I8Epi &e, hipStream_t st)
{
    return e.act == 0 ? linear_launch<BM, BN, WR, WC, NST, FLOW, 0>(x, ldx, w, Kp, M, N, e, st)
         : e.act == 1 ? linear_launch<BM, BN, WR, WC, NST, FLOW, 1>(x, ldx, w, Kp, M, N, e, st) : linear_launch<BM, BN, WR, WC, NST, FLOW, 2>(x, ldx, w, Kp, M, N, e, st);
}

template <int BM, int BN, int WR, int WC, int NST, bool FLOW, int ACT>
int requant_launch(const int8_t *x, long long ldx, const int8_t *w, int Kp, int M, int N, const I8Epi &e, hipStream_t st)
{
    typedef I8Tile<BM, BN, WR, WC, NST> T;
    constexpr int LDS = I8Requant<BM, BN, WC, NST * T::STAGE, FLOW>::LDS;
    static_assert(LDS <= 160 * 1024, "");
    if (LDS > 65536) {
        const hipError_t rc = hipFuncSetAttribute((const void *)int8_requant_kernel<BM, BN, WR, WC, NST, FLOW, ACT>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (rc != hipSuccess) return (int)rc;
    }
    const int tiles = p2c_cdiv(M, BM), grid = FLOW && tiles > I8_CUS ? I8_CUS : tiles;
    hipLaunchKernelGGL((int8_requant_kernel<BM, BN, WR, WC, NST, FLOW, ACT>), dim3(grid), dim3(64 * WR * WC), LDS, st, x, w, ldx, Kp, M, N, e);
    P2C_LAUNCH_CHECK();
    return P2C_OK;
}
template <int BM, int BN, int WR, int WC, int NST, bool FLOW>
int requant_any(const int8_t *x, long long ldx, const int8_t *w, int Kp, int M, int N, const I8Epi &e, hipStream_t st)
{
    return e.act == 0 ? requant_launch<BM, BN, WR, WC, NST, FLOW, 0>(x, ldx, w, Kp, M, N, e, st)
         : e.act == 1 ? requant_launch<BM, BN, WR, WC, NST, FLOW, 1>(x, ldx, w, Kp, M, N, e, st) : requant_launch<BM, BN, WR, WC, NST, FLOW, 2>(x, ldx, w, Kp, M, N, e, st);
}

constexpr long long I8_MAX_LD = 1 << 22;       // (a tile's offsets have 32 bits)
constexpr long long I8_MAX_M = (1 << 30) - 64; // (tiles of 64 rows in workgroups of 256: a grid holds fewer than 2^32 threads)
bool i8_shape_bad(long long M, int K, int Kp) { return M < 0 || M > I8_MAX_M || K < 1 || K > 131072 || Kp < K || Kp % 64; }

}  // namespace

extern "C" int p2c_int8_padded(int K) { return K < 1 ? 0 : (K + 63) / 64 * 64; }
extern "C" int p2c_int8_padded_out(int N) { return N < 1 ? 0 : (N + 255) / 256 * 256; }
extern "C" int p2c_int8_few_supported(int M, int K) { return M >= 1 && M <= 32 && K >= 1 && K <= 2048; }
// (the epilogue's softplus has no linear region of its own: above beta x = 17 it is the identity in 32 bits anyway, so the threshold has to lie there)
// The epilogue works in units of log2(e) / beta, and its rows have to keep their normal range there: beta >= 0.7 (unit >= 1; checked at the entry).
extern "C" int p2c_int8_requant_supported(int N, int act, float thr) { return N >= 1 && N <= 512 && (act != 2 || thr >= 17.0f); }

extern "C" int p2c_quantize_rows_at_once(int K) { return K < 1 ? 0 : quantize_rows_at_once(p2c_int8_padded(K)); }

extern "C" int p2c_quantize_rows(const void *x, int dtype, long long ldx, int M, int K, int Kp, int8_t *q, float *scale, void *stream)
{
    if (i8_shape_bad(M, K, Kp) || dtype < 0 || dtype > 2 || ldx < 0) return P2C_EINVAL;
    if (M == 0) return P2C_OK;
    if (!x || !q || !scale) return P2C_EINVAL;
    if ((uintptr_t)q & 15) return P2C_EALIGN;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == 0) return quantize_launch<Q_F32>(x, ldx, M, K, Kp, q, scale, st);
    if (dtype == 1) return quantize_launch<Q_BF16>(x, ldx, M, K, Kp, q, scale, st);
    return quantize_launch<Q_F16>(x, ldx, M, K, Kp, q, scale, st);
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
    return P2C_OK;
}

extern "C" int p2c_int8_linear(const int8_t *xq, long long ldx, const float *sx, const int8_t *wq, const float *sw, const float *bias, const float *add,
                               long long ldadd, int act, float beta, float thr, void *out, long long ldo, int dtype, int M, int N, int K, int Kp, void *stream)
{
    if (i8_shape_bad(M, K, Kp) || N < 1 || N > (1 << 20) || ldx < Kp || ldx > I8_MAX_LD) return P2C_EINVAL;
    I8Epi e;
    const int rc = i8_epilogue(e, sx, sw, bias, add, ldadd, act, beta, thr, out, ldo, dtype, N);
    if (rc != P2C_OK) return rc;
    if (M == 0) return P2C_OK;
    if (!xq || !sx || !wq || !sw || !out) return P2C_EINVAL;
    if (((uintptr_t)xq & 15) || ((uintptr_t)wq & 15) || ldx % 16) return P2C_EALIGN;
    const hipStream_t st = (hipStream_t)stream;
    // 256 x 256 reads each operand half as often as 128 x 128 (16384 x 4096 x 4096: 270 us against 384; 262144 x 512 x 512: 142 against 153), but has to
    // fill most of the 256 CUs; the same limit for 128 x 128 against 64 x 64.  From two tiles per CU on, one workgroup takes them one after the other
    // (16384 x 4096 x 4096: 278 -> 267 us; k-tiles for all three stages needed).  All of these from 20 calls out of idle, both forms in turn; in a long run of
    // calls, at its clock, the product of 16384 x 4096 x 4096 takes 236 us = 2330 TOP/s and that of 262144 x 512 x 512 136.
    const long long t256 = (long long)p2c_cdiv(M, 256) * p2c_cdiv(N, 256);
    if (t256 >= 2 * I8_CUS && Kp >= 192) return linear_any<256, 256, 2, 4, 3, true>(xq, ldx, wq, Kp, M, N, e, st);
    if (t256 >= 192) return linear_any<256, 256, 2, 4, 3, false>(xq, ldx, wq, Kp, M, N, e, st);
    if ((long long)p2c_cdiv(M, 128) * p2c_cdiv(N, 128) >= 192) return linear_any<128, 128, 2, 2, 3, false>(xq, ldx, wq, Kp, M, N, e, st);
    return linear_any<64, 64, 2, 2, 4, false>(xq, ldx, wq, Kp, M, N, e, st);
}

extern "C" int p2c_int8_linear_requant(const int8_t *xq, long long ldx, const float *sx, const int8_t *wq, const float *sw, const float *bias,
                                       const float *add, long long ldadd, int act, float beta, float thr, int8_t *out, int ldo, float *so, int M, int N, int K,
                                       int Kp, void *stream)
{
    if (i8_shape_bad(M, K, Kp) || !p2c_int8_requant_supported(N, act, thr) || (act == 2 && !(beta >= 0.7f)) || ldx < Kp || ldx > I8_MAX_LD || ldo != (N + 63) / 64 * 64) return P2C_EINVAL;
    I8Epi e;
    const int rc = i8_epilogue(e, sx, sw, bias, add, ldadd, act, beta, thr, out, ldo, 0, N);
    if (rc != P2C_OK) return rc;
    if (M == 0) return P2C_OK;
    if (!xq || !sx || !wq || !sw || !out || !so) return P2C_EINVAL;
    if (((uintptr_t)xq & 15) || ((uintptr_t)wq & 15) || ((uintptr_t)out & 15) || ldx % 16) return P2C_EALIGN;
    e.so = so;
    const hipStream_t st = (hipStream_t)stream;
    if (N <= 256) return requant_any<64, 256, 1, 4, 3, false>(xq, ldx, wq, Kp, M, N, e, st);
    // (two tiles per CU at least; k-tiles for both stages)
    if (p2c_cdiv(M, 128) >= 2 * I8_CUS && Kp >= 128) return requant_any<128, 512, 2, 4, 2, true>(xq, ldx, wq, Kp, M, N, e, st);
    return requant_any<64, 512, 1, 4, 2, false>(xq, ldx, wq, Kp, M, N, e, st);
}

extern "C" int p2c_int8_linear_few(const void *x, int xdtype, long long ldx, const int8_t *wq, const float *sw, const float *bias, const float *add,
                                   long long ldadd, int act, float beta, float thr, void *out, long long ldo, int dtype, int M, int N, int K, int Kp,
                                   void *stream)
{
    if (i8_shape_bad(M, K, Kp) || !p2c_int8_few_supported(M, K) || Kp > 2048 || N < 1 || N > (1 << 20) || xdtype < 0 || xdtype > 2 || ldx < 0) return P2C_EINVAL;
    I8Epi e;
    const int rc = i8_epilogue(e, nullptr, sw, bias, add, ldadd, act, beta, thr, out, ldo, dtype, N);
    if (rc != P2C_OK) return rc;
    if (!x || !wq || !sw || !out) return P2C_EINVAL;
    if ((uintptr_t)wq & 15) return P2C_EALIGN;
    const int lds = 32 * (Kp + 16) + 32 * 4 + 4 * 32 * 36 * 4;
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

// x as floats: quantised into ws (M * Kp bytes of rows, M scales behind them) on the way.  One call for both launches: at a few hundred rows the host's
// time is what a call costs (300 x 512 x 512: 18 us as two calls, 13 as one).
extern "C" int p2c_int8_linear_float(const void *x, int xdtype, long long ldx, const int8_t *wq, const float *sw, const float *bias, const float *add,
                                     long long ldadd, int act, float beta, float thr, void *out, long long ldo, int dtype, int M, int N, int K, int Kp,
                                     void *ws, void *stream)
{
    if (p2c_int8_few_supported(M, K)) return p2c_int8_linear_few(x, xdtype, ldx, wq, sw, bias, add, ldadd, act, beta, thr, out, ldo, dtype, M, N, K, Kp, stream);
    float *sx = reinterpret_cast<float *>(reinterpret_cast<int8_t *>(ws) + (long long)M * Kp);
    const int rc = p2c_int8_linear(nullptr, Kp, nullptr, nullptr, nullptr, bias, add, ldadd, act, beta, thr, nullptr, ldo, dtype, 0, N, K, Kp, stream);     // (the shapes, before anything is launched)
    if (rc != P2C_OK) return rc;
    if (M && (!ws || !wq || !sw || !out)) return P2C_EINVAL;
    if ((uintptr_t)wq & 15) return P2C_EALIGN;
    const int rq = p2c_quantize_rows(x, xdtype, ldx, M, K, Kp, (int8_t *)ws, sx, stream);
    return rq != P2C_OK ? rq : p2c_int8_linear((const int8_t *)ws, Kp, sx, wq, sw, bias, add, ldadd, act, beta, thr, out, ldo, dtype, M, N, K, Kp, stream);
}

extern "C" int p2c_int8_linear_requant_float(const void *x, int xdtype, long long ldx, const int8_t *wq, const float *sw, const float *bias, const float *add,
                                             long long ldadd, int act, float beta, float thr, int8_t *out, int ldo, float *so, int M, int N, int K, int Kp,
                                             void *ws, void *stream)
{
    float *sx = reinterpret_cast<float *>(reinterpret_cast<int8_t *>(ws) + (long long)M * Kp);
    const int rc = p2c_int8_linear_requant(nullptr, Kp, nullptr, nullptr, nullptr, bias, add, ldadd, act, beta, thr, nullptr, ldo, nullptr, 0, N, K, Kp, stream);
    if (rc != P2C_OK) return rc;
    if (M && (!ws || !wq || !sw || !out || !so)) return P2C_EINVAL;
    if (((uintptr_t)wq & 15) || ((uintptr_t)out & 15)) return P2C_EALIGN;
    const int rq = p2c_quantize_rows(x, xdtype, ldx, M, K, Kp, (int8_t *)ws, sx, stream);
    return rq != P2C_OK ? rq : p2c_int8_linear_requant((const int8_t *)ws, Kp, sx, wq, sw, bias, add, ldadd, act, beta, thr, out, ldo, so, M, N, K, Kp, stream);
}
