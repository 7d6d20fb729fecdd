// muon.hip -- Newton-Schulz orthogonalisation of matrices and the optimizer step around it (gfx950 only).
//
// X_0 = G / (|G|_F + eps), small side first (m x n, m <= n); then `steps` times   X <- a X + (b A + c A^2) X   with A = X X^T.
// The odd polynomial a s + b s^3 + c s^5 acts on every singular value, so X approaches the orthogonal factor of G.
//
// Precision: the iteration amplifies what a rounding leaves in the weak directions by up to a^steps (480 for five steps of 3.4445), so operands
// of 8 or 11 bits do not carry a 32-bit gradient (measured on matrices with decaying spectra: 1e-3 to 1e-1).  Every operand is held as TWO
// fp16 numbers, x 2^12 = hi + lo (22 - 23 bits), a product is hi hi + hi lo + lo hi in 32-bit sums on v_mfma_f32_32x32x16_f16: the error of a
// 32-bit product at a third of the fp16 rate, 5 times the rate of the chip's 32-bit matrix instruction.  2^12 fits because every matrix of
// the iteration is bounded by a small spectral norm (the host refuses coefficients that leave (0, 15)); what drops below the fp16 range is
// < 2^-37 of one.
// a X is added in the epilogue in 32 bits and not folded into the polynomial's diagonal: folded, the rounding of a + ... hits the weak
// directions (3.7e-5 against 1.3e-5 on a low-rank 512 x 512 gradient; 1.1e-5 for plain 32-bit arithmetic).
//
// Layout: X is kept twice, S = X [mP][nP] and T = X^T [nP][mP], so that all three products of a step are C[i][j] = sum_k P[i][k] Q[j][k] with
// k contiguous: A = S S^T, B = bA + cA A^T, T' = aT + T B^T (A, B symmetric: only tiles on and above the diagonal are computed, the mirror image
// is stored with them).  An element is 4 bytes, 8 consecutive k = 16 bytes of hi and 16 bytes of lo; sides are padded with zeros to the tile.
// All matrices of a call go through each product together: one launch per product, whatever their number (descriptors ride in the kernel
// arguments: no device table, capturable).  Matrices whose small side is <= 32 take ns_small_kernel: one workgroup each.
#include "tile_dma.h"
#include <math.h>

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));

constexpr int NS_MAX = 24;              // matrices per launch: 24 descriptors + the tile prefix stay under 4 KB of kernel arguments
constexpr int NS_SMALL = 32;            // small sides up to here take ns_small_kernel
constexpr int NS_SLABS = 64;            // partial sums of squares per matrix
constexpr float NS_SCALE = 4096.0f, NS_INV = 1.0f / 4096.0f;

struct NsMat {
    const char *src; float *mom; char *dst;
    long long src_rs, src_cs, src_bs, dst_rs, dst_cs, dst_bs;       // elements
    unsigned long long ws, ws_bs;                                   // bytes: workspace of batch entry 0, and to the next
    int m, n, mP, nP, batch, tall;                                  // tall: the small side runs along the columns
    float scale, decay;
};
struct NsArgs {
    char *ws;
    int nmat, dtype;                    // dtype of src and dst: 0 fp32, 1 bf16, 2 fp16
    float mu;                           // momentum (muon)
    int muon;                           // 0 orthogonalise, 1 momentum, 2 Nesterov momentum
    double eps;
    int start[NS_MAX + 1];              // first workgroup of each matrix in this launch
    NsMat mat[NS_MAX];
};

// workspace of one matrix: partial sums | S | T0 | T1 | A | B
__host__ __device__ __forceinline__ size_t ns_xbytes(int mP, int nP) { return (size_t)mP * nP * 4; }
__device__ __forceinline__ char *ns_S(char *w) { return w + NS_SLABS * 8; }
__device__ __forceinline__ char *ns_T(char *w, const NsMat &d, int which) { return ns_S(w) + (size_t)(1 + which) * ns_xbytes(d.mP, d.nP); }
__device__ __forceinline__ char *ns_A(char *w, const NsMat &d) { return ns_S(w) + 3 * ns_xbytes(d.mP, d.nP); }
__device__ __forceinline__ char *ns_B(char *w, const NsMat &d) { return ns_A(w, d) + ns_xbytes(d.mP, d.mP); }

__device__ __forceinline__ float ns_get(const char *p, long long i, int dt)
{
    if (dt == 0) return reinterpret_cast<const float *>(p)[i];
    if (dt == 1) return __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(p)[i] << 16);
    return (float)reinterpret_cast<const _Float16 *>(p)[i];
}
__device__ __forceinline__ void ns_put(char *p, long long i, int dt, float v)
{
    if (dt == 0) reinterpret_cast<float *>(p)[i] = v;
    else if (dt == 1) reinterpret_cast<__bf16 *>(p)[i] = (__bf16)v;
    else reinterpret_cast<_Float16 *>(p)[i] = (_Float16)v;
}

// u of element (i of the small side, j of the long side); first: the momentum is advanced, else the advanced one is read
__device__ __forceinline__ float ns_update_in(const NsArgs &a, const NsMat &d, int b, int i, int j, bool first)
{
    const long long r = d.tall ? j : i, c = d.tall ? i : j;
    const float g = ns_get(d.src, b * d.src_bs + r * d.src_rs + c * d.src_cs, a.dtype);
    if (!a.muon) return g;
    float *mp = d.mom + r * (d.tall ? d.m : d.n) + c;
    float mv = *mp;
    if (first) {
        mv = __builtin_fmaf(a.mu, mv, (1.0f - a.mu) * g);
        *mp = mv;
    }
    return a.muon == 2 ? __builtin_fmaf(a.mu, mv, (1.0f - a.mu) * g) : mv;
}

// O's element (i, j): stored, or taken off the parameter
__device__ __forceinline__ void ns_update_out(const NsArgs &a, const NsMat &d, int b, int i, int j, float o)
{
    const long long r = d.tall ? j : i, c = d.tall ? i : j;
    const long long at = b * d.dst_bs + r * d.dst_rs + c * d.dst_cs;
    if (!a.muon) { ns_put(d.dst, at, a.dtype, o); return; }
    float *p = reinterpret_cast<float *>(d.dst) + at;
    *p = *p * d.decay - d.scale * o;
}

// workgroup -> (matrix, batch entry, tile of it); everything uniform
__device__ __forceinline__ int ns_find(const NsArgs &a, int id)
{
    int i = 0;
    while (i + 1 < a.nmat && id >= a.start[i + 1]) ++i;
    return i;
}

__device__ __forceinline__ void ns_split8(const float *v, h16x8 &hi, h16x8 &lo)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        hi[e] = (_Float16)v[e];
        lo[e] = (_Float16)(v[e] - (float)hi[e]);
    }
}

// ---- sums of squares (64 bits: any 32-bit gradient fits), the momentum on the way.  NS_SLABS workgroups per matrix at most
__global__ void __launch_bounds__(256) ns_norm_kernel(const NsArgs a)
{
    __shared__ double red[4];
    const int mi = ns_find(a, blockIdx.x);
    const NsMat &d = a.mat[mi];
    const int slabs = (a.start[mi + 1] - a.start[mi]) / d.batch, t = blockIdx.x - a.start[mi], b = t / slabs, slab = t - b * slabs;
    const uint32_t total = (uint32_t)((long long)d.m * d.n), cols = d.tall ? d.m : d.n;     // at most 2^31
    double s = 0.0;
    for (uint32_t e = slab * 256 + threadIdx.x; e < total; e += slabs * 256) {
        const int r = (int)(e / cols), c = (int)(e - r * cols);
        const double u = ns_update_in(a, d, b, d.tall ? c : r, d.tall ? r : c, true);
        s += u * u;
    }
    s = p2c_wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) reinterpret_cast<double *>(a.ws + d.ws + b * d.ws_bs)[slab] = red[0] + red[1] + red[2] + red[3];
}

// ---- X_0: a 64 x 64 tile normalised and stored as S and T.  nslabs: of ns_norm_kernel's launch
__global__ void __launch_bounds__(256) ns_begin_kernel(const NsArgs a, const int max_slabs)
{
    __shared__ float x[64][65];
    __shared__ double part[NS_SLABS];
    const int mi = ns_find(a, blockIdx.x);
    const NsMat &d = a.mat[mi];
    const int ti = d.mP / 64, tj = d.nP / 64, t = blockIdx.x - a.start[mi], b = t / (ti * tj), tt = t - b * (ti * tj);
    const int i0 = tt / tj * 64, j0 = tt % tj * 64, tid = threadIdx.x;
    char *w = a.ws + d.ws + b * d.ws_bs;
    const int slabs = (int)min((long long)max_slabs, ((long long)d.m * d.n + 1023) / 1024);
    if (tid < slabs) part[tid] = reinterpret_cast<const double *>(w)[tid];
    __syncthreads();
    double s = 0.0;
    for (int k = 0; k < slabs; ++k) s += part[k];
    const double inv = (double)NS_SCALE / (sqrt(s) + a.eps);
#pragma unroll 4
    for (int q = 0; q < 16; ++q) {
        const int e = tid + 256 * q, u = e >> 6, v = e & 63;
        const int i = d.tall ? v : u, j = d.tall ? u : v;
        x[i][j] = (i0 + i < d.m && j0 + j < d.n) ? (float)((double)ns_update_in(a, d, b, i0 + i, j0 + j, false) * inv) : 0.f;
    }
    __syncthreads();
    char *S = ns_S(w), *T = ns_T(w, d, 0);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int e = tid + 256 * q, r = e >> 3, c8 = (e & 7) * 8;
        float v[8];
        h16x8 hi, lo;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = x[r][c8 + k];
        ns_split8(v, hi, lo);
        h16x8 *o = reinterpret_cast<h16x8 *>(S + ((size_t)(i0 + r) * d.nP + j0 + c8) * 4);
        o[0] = hi; o[1] = lo;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = x[c8 + k][r];
        ns_split8(v, hi, lo);
        o = reinterpret_cast<h16x8 *>(T + ((size_t)(j0 + r) * d.mP + i0 + c8) * 4);
        o[0] = hi; o[1] = lo;
    }
}

// tile t of the upper triangle of an nt x nt grid, row by row -> (i, j), j >= i
__device__ __forceinline__ void ns_triangle(int t, int nt, int &i, int &j)
{
    i = 0;
    while (t >= nt - i) { t -= nt - i; ++i; }
    j = i + t;
}

// ---- one product of a step for every matrix.  PH 1: A = S S^T.  2: B = b A + c A A^T.  3: T' = a T + T B^T (and S').  4: as 3, into the result.
// Tile TB x TB, four waves of TB/2 x TB/2, k-tiles of 32 (128 bytes a row) in NST LDS stages filled by direct copies, one barrier per k-tile.
template <int TB, int NST, int PH>
__global__ void __launch_bounds__(256) ns_product_kernel(const NsArgs a, const float ca, const float cb, const int cur)
{
    constexpr int RB = 128, STAGE = 2 * TB * RB, NT = TB / 64, LPW = 2 * TB * RB / 1024 / 4;
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int mi = ns_find(a, blockIdx.x);
    const NsMat &d = a.mat[mi];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), il = lane & 31, h = lane >> 5;
    const int mt = d.mP / TB, per = PH <= 2 ? mt * (mt + 1) / 2 : mt * (d.nP / TB);
    int t = blockIdx.x - a.start[mi];
    const int b = t / per;
    t -= b * per;
    int ti, tj;                                     // tile rows of P and of Q
    if (PH <= 2) ns_triangle(t, mt, ti, tj);
    else { ti = t / mt; tj = t - ti * mt; }
    char *w = a.ws + d.ws + b * d.ws_bs;
    const char *P, *Q;
    int K;
    if (PH == 1) { P = Q = ns_S(w); K = d.nP; }
    else if (PH == 2) { P = Q = ns_A(w, d); K = d.mP; }
    else { P = ns_T(w, d, cur); Q = ns_B(w, d); K = d.mP; }
    const long long ld = (long long)K * 4;
    P += (long long)ti * TB * ld;
    Q += (long long)tj * TB * ld;
    const int KT = K / 32;

    f32x16 acc[NT][NT];
#pragma unroll
    for (int p = 0; p < NT; ++p)
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[p][q][r] = 0.f;

#define P2C_NS_COPY(KT_)                                                                             \
    do {                                                                                             \
        const int k__ = min((KT_), KT - 1);                                                          \
        char *st__ = smem + ((KT_) % NST) * STAGE;                                                   \
        p2c_tile_copy<TB, RB, 4>(P + (long long)k__ * RB, ld, TB - 1, st__, wave, lane);             \
        p2c_tile_copy<TB, RB, 4>(Q + (long long)k__ * RB, ld, TB - 1, st__ + TB * RB, wave, lane);   \
    } while (0)
#pragma unroll
    for (int s = 0; s < NST - 1; ++s) P2C_NS_COPY(s);
    const int wr = (wave >> 1) * (TB / 2), wc = (wave & 1) * (TB / 2);
    for (int kt = 0; kt < KT; ++kt) {
        p2c_tile_wait<(NST - 2) * LPW>();           // stage kt is here, and nobody reads stage kt - 1 any more
        P2C_NS_COPY(kt + NST - 1);                  // (past the end: the last tile again, into a stage that is never read: the count in flight stays exact)
        const char *ps = smem + (kt % NST) * STAGE, *qs = ps + TB * RB;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            h16x8 p[NT][2], q[NT][2];
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) {
                    const int c = (2 * s + h) * 2 + pl;
                    p[x][pl] = *reinterpret_cast<const h16x8 *>(ps + p2c_tile_at<RB>(wr + x * 32 + il, c));
                    q[x][pl] = *reinterpret_cast<const h16x8 *>(qs + p2c_tile_at<RB>(wc + x * 32 + il, c));
                }
#pragma unroll
            for (int pr = 0; pr < 3; ++pr)          // small products first
#pragma unroll
                for (int x = 0; x < NT; ++x)
#pragma unroll
                    for (int y = 0; y < NT; ++y)
                        acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(p[x][pr == 1], q[y][pr == 0], acc[x][y], 0, 0, 0);
        }
    }
#undef P2C_NS_COPY
    p2c_tile_wait<0>();                             // the surplus copies have landed: the stages are free

    // ---- epilogue.  A lane holds column il of a 32 x 32 piece, rows 8 g + 4 h + (0..3): four consecutive k of the transposed image, which is
    // read (the addend) and written from the registers; the straight image goes through LDS to get 8 consecutive k per lane.
    float *stage = reinterpret_cast<float *>(smem) + wave * (32 * 36);
    const bool mirror = PH == 3 || (PH <= 2 && ti != tj);
    char *o1 = PH == 1 ? ns_A(w, d) : PH == 2 ? ns_B(w, d) : ns_T(w, d, cur ^ 1);
    char *o2 = PH == 3 || PH == 4 ? ns_S(w) : o1;
    const char *old = PH == 2 ? ns_A(w, d) : ns_S(w);
    const int ld1 = d.mP, ld2 = PH <= 2 ? d.mP : d.nP;
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int y = 0; y < NT; ++y) {
            const int r0 = ti * TB + wr + x * 32, c0 = tj * TB + wc + y * 32, col = c0 + il;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const size_t at2 = ((size_t)col * ld2 + r0 + 8 * g) * 4 + 8 * h;
                float v[4];
                if (PH == 1) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = acc[x][y][4 * g + e] * NS_INV;
                } else {
                    const h16x4 oh = *reinterpret_cast<const h16x4 *>(old + at2), ol = *reinterpret_cast<const h16x4 *>(old + at2 + 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(ca, (float)oh[e] + (float)ol[e], cb * (acc[x][y][4 * g + e] * NS_INV));
                }
                if (PH == 4) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = col, j = r0 + 8 * g + 4 * h + e;
                        if (i < d.m && j < d.n) ns_update_out(a, d, b, i, j, v[e] * NS_INV);
                    }
                } else {
                    if (mirror) {
                        h16x4 vh, vl;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            vh[e] = (_Float16)v[e];
                            vl[e] = (_Float16)(v[e] - (float)vh[e]);
                        }
                        *reinterpret_cast<h16x4 *>(o2 + at2) = vh;
                        *reinterpret_cast<h16x4 *>(o2 + at2 + 16) = vl;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) stage[(8 * g + 4 * h + e) * 36 + il] = v[e];
                }
            }
            if (PH != 4) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const int u = lane + 64 * q, r = u >> 2, c8 = (u & 3) * 8;
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = stage[r * 36 + c8 + k];
                    h16x8 hi, lo;
                    ns_split8(v, hi, lo);
                    h16x8 *o = reinterpret_cast<h16x8 *>(o1 + ((size_t)(r0 + r) * ld1 + c0 + c8) * 4);
                    o[0] = hi; o[1] = lo;
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        }
}

// ---- small side <= 32: one workgroup per matrix, in the m x m space and in 64 bits.  X_k = Q_k X_0 with Q and A polynomials of A_0 = X_0 X_0^T:
// q = a + bA + cA^2, Q <- q Q, A <- q A q.  G is read twice and nothing else moves.  64 bits are what this form needs (A holds SQUARED singular
// values and a rounding grows by a^2 per step: 2.5e5 over five); at this size they cost less than the launches of the tiled form.
// coefficients: [steps][3] in constant order a, b, c
struct NsCoef { int steps; float c[16][3]; };

__device__ __forceinline__ double ns_dot(const double (*x)[NS_SMALL + 1], const double (*y)[NS_SMALL + 1], int i, int j, int m)
{
    double s = 0.0;
    for (int k = 0; k < m; ++k) s = fma(x[i][k], y[k][j], s);
    return s;
}

__global__ void __launch_bounds__(256) ns_small_kernel(const NsArgs a, const NsCoef co)
{
    __shared__ double A[NS_SMALL][NS_SMALL + 1], Q[NS_SMALL][NS_SMALL + 1], U[NS_SMALL][NS_SMALL + 1], V[NS_SMALL][NS_SMALL + 1];
    __shared__ float x[NS_SMALL][65];
    const int mi = ns_find(a, blockIdx.x);
    const NsMat &d = a.mat[mi];
    const int b = blockIdx.x - a.start[mi], tid = threadIdx.x, m = d.m, n = d.n;
    const int pi = tid >> 4, pj = tid & 15;                     // this thread's 2 x 2 entries of an m x m matrix
    double g[2][2] = {{0.0, 0.0}, {0.0, 0.0}};
    const int tasks = m * 64;
    // 64 long indices at a time, the next ones in flight under the sums
    float nx[8];
    auto fetch = [&](int j0, bool first) {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int e = tid + 256 * q;
            const int i = d.tall ? e % m : e >> 6, j = j0 + (d.tall ? e / m : e & 63);
            nx[q] = (e < tasks && j < n) ? ns_update_in(a, d, b, i, j, first) : 0.f;
        }
    };
    auto place = [&]() {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int e = tid + 256 * q;
            if (e < tasks) x[d.tall ? e % m : e >> 6][d.tall ? e / m : e & 63] = nx[q];
        }
    };
    fetch(0, true);
    for (int j0 = 0; j0 < n; j0 += 64) {
        __syncthreads();
        place();
        __syncthreads();
        if (j0 + 64 < n) fetch(j0 + 64, true);
        if (2 * pi < m && 2 * pj < m) {
            const int i1 = min(2 * pi + 1, m - 1), k1 = min(2 * pj + 1, m - 1);
#pragma unroll 4
            for (int j = 0; j < 64; ++j) {
                const double u0 = x[2 * pi][j], u1 = x[i1][j], v0 = x[2 * pj][j], v1 = x[k1][j];
                g[0][0] = fma(u0, v0, g[0][0]);
                g[0][1] = fma(u0, v1, g[0][1]);
                g[1][0] = fma(u1, v0, g[1][0]);
                g[1][1] = fma(u1, v1, g[1][1]);
            }
        }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < 2; ++q)
            if (2 * pi + p < m && 2 * pj + q < m) A[2 * pi + p][2 * pj + q] = g[p][q];
    __syncthreads();
    double tr = 0.0;
    for (int k = 0; k < m; ++k) tr += A[k][k];
    const double inv = 1.0 / (sqrt(tr) + a.eps);
    __syncthreads();
    for (int e = tid; e < m * m; e += 256) {
        const int i = e / m, j = e - i * m;
        A[i][j] *= inv * inv;
        Q[i][j] = i == j ? inv : 0.0;                           // the normalisation of X_0 rides in Q
    }
    __syncthreads();
    for (int s = 0; s < co.steps; ++s) {
        const double c0 = co.c[s][0], c1 = co.c[s][1], c2 = co.c[s][2];
        for (int e = tid; e < m * m; e += 256) {
            const int i = e / m, j = e - i * m;
            U[i][j] = c2 * ns_dot(A, A, i, j, m) + c1 * A[i][j] + (i == j ? c0 : 0.0);      // q
        }
        __syncthreads();
        for (int e = tid; e < m * m; e += 256) V[e / m][e % m] = ns_dot(U, Q, e / m, e % m, m);
        __syncthreads();
        for (int e = tid; e < m * m; e += 256) Q[e / m][e % m] = V[e / m][e % m];
        if (s + 1 == co.steps) break;
        __syncthreads();
        for (int e = tid; e < m * m; e += 256) V[e / m][e % m] = ns_dot(U, A, e / m, e % m, m);
        __syncthreads();
        for (int e = tid; e < m * m; e += 256) A[e / m][e % m] = ns_dot(V, U, e / m, e % m, m);
        __syncthreads();
    }
    fetch(0, false);
    for (int j0 = 0; j0 < n; j0 += 64) {
        __syncthreads();
        place();
        __syncthreads();
        if (j0 + 64 < n) fetch(j0 + 64, false);
        for (int e = tid; e < tasks; e += 256) {
            const int i = e >> 6, j = e & 63;
            if (j0 + j < n) {
                double s = 0.0;
                for (int k = 0; k < m; ++k) s = fma(Q[i][k], (double)x[k][j], s);
                ns_update_out(a, d, b, i, j0 + j, (float)s);
            }
        }
    }
}

inline int ns_pad(int v, int to) { return (v + to - 1) / to * to; }
inline bool ns_is_small(const p2c_ns_matrix &m) { return (m.rows < m.cols ? m.rows : m.cols) <= NS_SMALL; }

// Tile of a chunk's products: 128 keeps the matrix units busy (a wave reads 16 KB of operands for 24 instructions), 64 has four times the
// workgroups and a shorter chain per workgroup.
inline int ns_tile(const p2c_ns_matrix *mats, int n)
{
    long long t128 = 0;
    for (int i = 0; i < n; ++i)
        if (!ns_is_small(mats[i])) {
            const int s = mats[i].rows < mats[i].cols ? mats[i].rows : mats[i].cols;
            const long long mt = (s + 127) / 128;
            t128 += mt * (mt + 1) / 2 * mats[i].batch;
        }
    return t128 >= 256 ? 128 : 64;
}

inline size_t ns_one_ws(const p2c_ns_matrix &m, int tile)
{
    if (ns_is_small(m)) return 0;
    const int s = m.rows < m.cols ? m.rows : m.cols, l = m.rows < m.cols ? m.cols : m.rows, mP = ns_pad(s, tile), nP = ns_pad(l, tile);
    return NS_SLABS * 8 + 3 * ns_xbytes(mP, nP) + 2 * ns_xbytes(mP, mP);
}

int ns_check(const p2c_ns_matrix *mats, int n)
{
    if (!mats || n <= 0) return P2C_EINVAL;
    for (int i = 0; i < n; ++i)
        if (mats[i].rows < 0 || mats[i].cols < 0 || mats[i].batch < 0 || mats[i].rows > (1 << 20) || mats[i].cols > (1 << 20) ||
            (long long)mats[i].rows * mats[i].cols > (1ll << 31) || mats[i].batch > (1 << 16)) return P2C_EINVAL;
    return P2C_OK;
}

inline size_t ns_chunk_ws(const p2c_ns_matrix *mats, int n)
{
    const int tile = ns_tile(mats, n);
    size_t s = 0;
    for (int i = 0; i < n; ++i) s += ns_one_ws(mats[i], tile) * mats[i].batch;
    return s;
}

template <int TB, int NST>
int ns_products(NsArgs &a, const NsCoef &co, int total_sym, int total_all, const int *sym, const int *all, hipStream_t st)
{
    constexpr int LDS = 2 * TB * 128 * NST;
    static_assert(LDS >= 4 * 32 * 36 * 4, "");
    for (int s = 0; s < co.steps; ++s) {
        const bool last = s + 1 == co.steps;
        for (int i = 0; i <= a.nmat; ++i) a.start[i] = sym[i];
        hipLaunchKernelGGL((ns_product_kernel<TB, NST, 1>), dim3(total_sym), dim3(256), LDS, st, a, 0.f, 1.f, s & 1);
        P2C_LAUNCH_CHECK();
        hipLaunchKernelGGL((ns_product_kernel<TB, NST, 2>), dim3(total_sym), dim3(256), LDS, st, a, co.c[s][1], co.c[s][2], s & 1);
        P2C_LAUNCH_CHECK();
        for (int i = 0; i <= a.nmat; ++i) a.start[i] = all[i];
        if (last) hipLaunchKernelGGL((ns_product_kernel<TB, NST, 4>), dim3(total_all), dim3(256), LDS, st, a, co.c[s][0], 1.f, s & 1);
        else hipLaunchKernelGGL((ns_product_kernel<TB, NST, 3>), dim3(total_all), dim3(256), LDS, st, a, co.c[s][0], 1.f, s & 1);
        P2C_LAUNCH_CHECK();
    }
    return P2C_OK;
}

int ns_chunk(const p2c_ns_matrix *mats, int n, int dtype, float mu, int muon, const NsCoef &co, double eps, char *ws, hipStream_t st)
{
    NsArgs a, sm;
    a.ws = ws; a.dtype = dtype; a.mu = mu; a.muon = muon; a.eps = eps; a.nmat = 0;
    sm = a;
    const int tile = ns_tile(mats, n);
    int slabs[NS_MAX + 1] = {0}, tiles[NS_MAX + 1] = {0}, sym[NS_MAX + 1] = {0}, all[NS_MAX + 1] = {0};
    size_t off = 0;
    sm.start[0] = 0;
    for (int i = 0; i < n; ++i) {
        const p2c_ns_matrix &q = mats[i];
        if (!q.rows || !q.cols || !q.batch) continue;           // nothing to do
        const bool small = ns_is_small(q);
        NsArgs &t = small ? sm : a;
        NsMat &d = t.mat[t.nmat];
        d.src = (const char *)q.src; d.mom = q.mom; d.dst = (char *)q.dst;
        d.src_rs = q.src_rs; d.src_cs = q.src_cs; d.src_bs = q.src_bs;
        d.dst_rs = q.dst_rs; d.dst_cs = q.dst_cs; d.dst_bs = q.dst_bs;
        d.tall = q.rows > q.cols;
        d.m = d.tall ? q.cols : q.rows; d.n = d.tall ? q.rows : q.cols;
        d.mP = ns_pad(d.m, tile); d.nP = ns_pad(d.n, tile);
        d.batch = q.batch; d.scale = q.scale; d.decay = q.decay;
        d.ws = off; d.ws_bs = ns_one_ws(q, tile);
        off += d.ws_bs * q.batch;
        const int k = t.nmat++;
        if (small) {
            sm.start[k + 1] = sm.start[k] + q.batch;
        } else {
            const long long sl = ((long long)d.m * d.n + 1023) / 1024;
            const int mt = d.mP / tile;
            slabs[k + 1] = slabs[k] + (int)(sl < NS_SLABS ? sl : NS_SLABS) * q.batch;
            tiles[k + 1] = tiles[k] + (d.mP / 64) * (d.nP / 64) * q.batch;
            sym[k + 1] = sym[k] + mt * (mt + 1) / 2 * q.batch;
            all[k + 1] = all[k] + mt * (d.nP / tile) * q.batch;
        }
    }
    if (sm.nmat) {
        hipLaunchKernelGGL(ns_small_kernel, dim3(sm.start[sm.nmat]), dim3(256), 0, st, sm, co);
        P2C_LAUNCH_CHECK();
    }
    if (!a.nmat) return P2C_OK;
    for (int i = 0; i <= a.nmat; ++i) a.start[i] = slabs[i];
    hipLaunchKernelGGL(ns_norm_kernel, dim3(slabs[a.nmat]), dim3(256), 0, st, a);
    P2C_LAUNCH_CHECK();
    for (int i = 0; i <= a.nmat; ++i) a.start[i] = tiles[i];
    hipLaunchKernelGGL(ns_begin_kernel, dim3(tiles[a.nmat]), dim3(256), 0, st, a, NS_SLABS);
    P2C_LAUNCH_CHECK();
    return tile == 128 ? ns_products<128, 2>(a, co, sym[a.nmat], all[a.nmat], sym, all, st)
                       : ns_products<64, 4>(a, co, sym[a.nmat], all[a.nmat], sym, all, st);
}

int ns_run(const p2c_ns_matrix *mats, int n, int dtype, float mu, int muon, int steps, const float *coeffs, double eps, void *ws, size_t ws_bytes,
           void *stream)
{
    const int rc = ns_check(mats, n);
    if (rc != P2C_OK) return rc;
    if (steps < 1 || steps > 16 || !coeffs || !(eps > 0.0) || dtype < 0 || dtype > 2) return P2C_EINVAL;
    NsCoef co;
    co.steps = steps;
    // every matrix of the iteration has to stay inside the range of the scaled fp16 pairs: follow the bound of the spectrum
    double top = 1.0;
    for (int s = 0; s < steps; ++s) {
        const double c0 = coeffs[3 * s], c1 = coeffs[3 * s + 1], c2 = coeffs[3 * s + 2];
        if (!isfinite(c0) || !isfinite(c1) || !isfinite(c2)) return P2C_EINVAL;
        double p = 0.0, q = 0.0;
        for (int k = 0; k <= 256; ++k) {
            const double x = top * k / 256, t = x * x, bb = c1 * t + c2 * t * t, qq = c0 + bb;
            p = fmax(p, fabs(x * qq));
            q = fmax(q, fmax(fabs(bb), fabs(c0)));
        }
        if (!(p < 3.8) || !(q < 15.0)) return P2C_EINVAL;
        top = 1.01 * p;
        for (int k = 0; k < 3; ++k) co.c[s][k] = coeffs[3 * s + k];
    }
    for (int s = steps; s < 16; ++s) co.c[s][0] = co.c[s][1] = co.c[s][2] = 0.f;
    for (int i = 0; i < n; ++i) {
        const p2c_ns_matrix &q = mats[i];
        if (q.rows && q.cols && q.batch && (!q.src || !q.dst || (muon && (!q.mom || q.batch != 1)))) return P2C_EINVAL;
    }
    size_t need = 0;
    for (int i = 0; i < n; i += NS_MAX) {
        const size_t c = ns_chunk_ws(mats + i, n - i < NS_MAX ? n - i : NS_MAX);
        need = c > need ? c : need;
    }
    if (need > ws_bytes || (need && (!ws || ((uintptr_t)ws & 15)))) return P2C_EINVAL;
    for (int i = 0; i < n; i += NS_MAX) {
        const int r = ns_chunk(mats + i, n - i < NS_MAX ? n - i : NS_MAX, dtype, mu, muon, co, eps, (char *)ws, (hipStream_t)stream);
        if (r != P2C_OK) return r;
    }
    return P2C_OK;
}

}  // namespace

extern "C" size_t p2c_newton_schulz_ws_bytes(const p2c_ns_matrix *mats_host, int n)
{
    if (ns_check(mats_host, n) != P2C_OK) return 0;
    size_t need = 0;
    for (int i = 0; i < n; i += NS_MAX) {
        const size_t c = ns_chunk_ws(mats_host + i, n - i < NS_MAX ? n - i : NS_MAX);
        need = c > need ? c : need;
    }
    return need;
}

extern "C" int p2c_newton_schulz(const p2c_ns_matrix *mats_host, int n, int dtype, int steps, const float *coeffs_host, double eps, void *ws,
                                 size_t ws_bytes, void *stream)
{
    return ns_run(mats_host, n, dtype, 0.f, 0, steps, coeffs_host, eps, ws, ws_bytes, stream);
}

extern "C" int p2c_muon_step_f32(const p2c_ns_matrix *mats_host, int n, float momentum, int nesterov, int steps, const float *coeffs_host,
                                 double eps, void *ws, size_t ws_bytes, void *stream)
{
    if (!(momentum >= 0.f && momentum < 1.f)) return P2C_EINVAL;
    return ns_run(mats_host, n, 0, momentum, nesterov ? 2 : 1, steps, coeffs_host, eps, ws, ws_bytes, stream);
}
