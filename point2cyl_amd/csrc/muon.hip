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
// < 2^-37 of one.  That floor is absolute where a 32-bit number's is relative, so the steps must not bring it up: the host refuses steps that amplify
// weak directions by more than 2^15 together (rows 1e-9 of the others, 64 x 128: 1.5e-6 off after 5 steps, 2.3e-6 after 8 = 2^14.3, plain 32-bit arithmetic 1.3e-6
// and 1.9e-6; after 10 it would be 1.0e-5 against 2.2e-6, after 16 1.7e-2 against 2.3e-6).
// a X is added to the finished product in 32 bits and not folded into the polynomial's diagonal: folded, the rounding of a + ... hits the weak
// directions (3.7e-5 against 1.3e-5 on a low-rank 512 x 512 gradient; 1.1e-5 for plain 32-bit arithmetic).
//
// Layout: X is kept twice, S = X (rows mP, k nP) and T = X^T (rows nP, k mP), so that all three products of a step are C[i][j] = sum_k P[i][k] Q[j][k]:
// A = S S^T, B = bA + cA A^T, T' = aT + T B^T (A, B symmetric: only tiles on and above the diagonal are computed, the mirror image
// is stored with them).  An element is 4 bytes, 8 consecutive k = 16 bytes of hi and 16 bytes of lo; an image is cut into blocks of
// 32 k, [k / 32][row][128 bytes]: what a tile needs of a block is one run of memory, and a 32 x 32 piece of a result is 4 KB of it.  Sides are padded
// with zeros to the tile.
// All matrices of a call go through each product together: one launch per product, whatever their number (the descriptors ride in the arguments of
// the first launch: no copy from the host, capturable).  Small ones (up to 16 rows) take ns_small, one workgroup each, where no larger ones are there to ride
// with.
#include "tile_dma.h"
#include <math.h>
#include <string.h>

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));

constexpr int NS_MAX = 24;              // matrices per chunk: the table stays under 4 KB of kernel arguments
constexpr int NS_SMALL = 16;            // small sides up to here can take ns_small
constexpr int NS_PARTS = 1024;          // partial sums of squares per matrix at most
constexpr float NS_SCALE = 4096.0f, NS_INV = 1.0f / 4096.0f;

struct NsMat {
    const char *src; float *mom; char *dst;
    long long src_rs, src_cs, src_bs, dst_rs, dst_cs, dst_bs;       // elements
    unsigned long long ws, ws_bs;                                   // bytes: workspace of batch entry 0, and to the next
    int m, n, mP, nP, batch, tall;                                  // tall: the small side runs along the columns
    float scale, decay;
};
enum { NS_NORM = 0, NS_TILES = 1, NS_SYM = 2, NS_ALL = 3 };
// The descriptors travel as an argument of the first launches; ns_begin_kernel leaves them in the workspace, with one record per workgroup of the
// products.  A product's chain of cold misses (nothing is in the caches when a kernel starts) is then ONE long before its operands are on their way:
// arguments preloaded into registers, record, copies.  Matrices [0, nbig) are tiled, [nbig, nbig + nsmall) small; start[phase][i]: first workgroup of
// matrix i.
struct NsTab {
    char *ws;
    int nbig, nsmall, dtype;            // dtype of src and dst: 0 fp32, 1 bf16, 2 fp16
    float mu;                           // momentum
    int muon;                           // 0 orthogonalise, 1 momentum, 2 Nesterov momentum
    double eps;
    int nsym, nall, tsym, tall;         // products: workgroups and tile of the symmetric ones, of the others
    int mid, unused;                    // every tiled matrix fits ns_mid_kernel
    int start[4][NS_MAX + 1];
    int small[NS_MAX + 1];
    NsMat mat[NS_MAX];
};
static_assert(sizeof(NsTab) % 4 == 0 && sizeof(NsTab) <= 3900, "with the coefficients within 4 KB of arguments");

struct NsRec { unsigned long long w; int ti, tj, mP, nP, mi, b; };      // a workgroup of a product: workspace of its matrix, tile rows of P and Q
static_assert(sizeof(NsRec) == 32, "");
constexpr size_t NS_TAB_BYTES = (sizeof(NsTab) + 511) / 512 * 512;
// workspace: table | records of the symmetric products, of the others | matrices
__host__ __device__ __forceinline__ size_t ns_head(int nsym, int nall) { return NS_TAB_BYTES + ((size_t)(nsym + nall) * sizeof(NsRec) + 511) / 512 * 512; }

// workspace of a matrix: partial sums | S | T0 | T1 | A | B
__host__ __device__ __forceinline__ size_t ns_xbytes(int mP, int nP) { return (size_t)mP * nP * 4; }
__device__ __forceinline__ char *ns_S(char *w) { return w + NS_PARTS * 8; }
template <class D> __device__ __forceinline__ char *ns_T(char *w, const D &d, int which) { return ns_S(w) + (size_t)(1 + which) * ns_xbytes(d.mP, d.nP); }
template <class D> __device__ __forceinline__ char *ns_A(char *w, const D &d) { return ns_S(w) + 3 * ns_xbytes(d.mP, d.nP); }
template <class D> __device__ __forceinline__ char *ns_B(char *w, const D &d) { return ns_A(w, d) + ns_xbytes(d.mP, d.mP); }

__device__ __forceinline__ const char *ns_src(const NsTab &a, const NsMat &d, int b) { return d.src + b * d.src_bs * (a.dtype == 0 ? 4 : 2); }

// What differs between calls (type, momentum) is decided once per group of N elements, so that their loads are in flight together: decided per element
// they wait for each other (32 of them: 14000 clocks).
// G of N elements: at(q) = offset in elements, always one of the matrix
template <int N, class At>
__device__ __forceinline__ void ns_load_n(const char *src, int dtype, float (&v)[N], At at)
{
    if (dtype == 0) {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = reinterpret_cast<const float *>(src)[at(q)];
    } else if (dtype == 1) {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(src)[at(q)] << 16);
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = (float)reinterpret_cast<const _Float16 *>(src)[at(q)];
    }
}
// u of N elements from G and the momentum; first: the momentum is advanced, else the advanced one is read.  at_m(q): its offset; ok(q): the element exists
template <int N, class At, class Ok>
__device__ __forceinline__ void ns_momentum_n(const NsTab &a, float *mom, float (&v)[N], bool first, At at_m, Ok ok)
{
    float m[N];
#pragma unroll
    for (int q = 0; q < N; ++q) m[q] = mom[at_m(q)];
    if (first) {
#pragma unroll
        for (int q = 0; q < N; ++q) m[q] = __builtin_fmaf(a.mu, m[q], (1.0f - a.mu) * v[q]);
#pragma unroll
        for (int q = 0; q < N; ++q)
            if (ok(q)) mom[at_m(q)] = m[q];
    }
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] = a.muon == 2 ? __builtin_fmaf(a.mu, m[q], (1.0f - a.mu) * v[q]) : m[q];
}
// N elements of the result: stored, or taken off the parameter.  i of the small side, j of the long one
template <int N, class I, class J>
__device__ __forceinline__ void ns_store_n(const NsTab &a, const NsMat &d, int b, const float (&o)[N], I i, J j)
{
    auto ok = [&](int q) { return i(q) < d.m && j(q) < d.n; };
    auto at = [&](int q) { return b * d.dst_bs + (d.tall ? j(q) : i(q)) * d.dst_rs + (d.tall ? i(q) : j(q)) * d.dst_cs; };
    if (a.muon) {
        float *p = reinterpret_cast<float *>(d.dst), v[N];
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = ok(q) ? p[at(q)] : 0.f;
#pragma unroll
        for (int q = 0; q < N; ++q)
            if (ok(q)) p[at(q)] = v[q] * d.decay - d.scale * o[q];
    } else if (a.dtype == 0) {
#pragma unroll
        for (int q = 0; q < N; ++q)
            if (ok(q)) reinterpret_cast<float *>(d.dst)[at(q)] = o[q];
    } else if (a.dtype == 1) {
#pragma unroll
        for (int q = 0; q < N; ++q)
            if (ok(q)) reinterpret_cast<__bf16 *>(d.dst)[at(q)] = (__bf16)o[q];
    } else {
#pragma unroll
        for (int q = 0; q < N; ++q)
            if (ok(q)) reinterpret_cast<_Float16 *>(d.dst)[at(q)] = (_Float16)o[q];
    }
}

// workgroup -> matrix; everything uniform
__device__ __forceinline__ int ns_find(const int *start, int n, int id)
{
    int i = 0;
    while (i + 1 < n && id >= start[i + 1]) ++i;
    return i;
}

// Consecutive workgroups go round the 8 XCDs; this order gives each XCD a contiguous eighth of a matrix' tiles instead, so that tiles that share
// operand rows share an L2 (8 x 1024 x 2048: 1662 -> 1557 us a call).  Per matrix and not over the whole list: whole matrices per XCD would leave XCDs
// with unequal work (a list of 2048 x 2048, 4000 x 1000, ...: 1579 -> 1764).
__device__ __forceinline__ int ns_xcd_order(int id, int grid)
{
    const int x = id & 7, q = grid >> 3, r = grid & 7;
    return x * q + min(x, r) + (id >> 3);
}

__device__ __forceinline__ void ns_split8(const float *v, h16x8 &hi, h16x8 &lo)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        hi[e] = (_Float16)v[e];
        lo[e] = (_Float16)(v[e] - (float)hi[e]);
    }
}

// 64 x 64 elements of a matrix in 16 registers a thread, 16 loads in flight: rows r0 + (tid >> 6) + 4 q, column c0 + (tid & 63); zeros outside
__device__ __forceinline__ void ns_load_tile(const NsTab &a, const NsMat &d, const char *src, int r0, int c0, bool first, float (&v)[16])
{
    const int rows = d.tall ? d.n : d.m, cols = d.tall ? d.m : d.n, r = r0 + (threadIdx.x >> 6), c = c0 + (threadIdx.x & 63), cc = min(c, cols - 1);
    auto ok = [&](int q) { return r + 4 * q < rows && c < cols; };
    ns_load_n(src, a.dtype, v, [&](int q) { return min(r + 4 * q, rows - 1) * d.src_rs + cc * d.src_cs; });
    if (a.muon) ns_momentum_n(a, d.mom, v, first, [&](int q) { return (long long)min(r + 4 * q, rows - 1) * cols + cc; }, ok);
#pragma unroll
    for (int q = 0; q < 16; ++q) v[q] = ok(q) ? v[q] : 0.f;
}

// what brings a matrix whose squares sum to s to unit norm.  A zero matrix stays zero whatever eps is (1 / eps may leave 64 bits); any other 32-bit matrix has a norm
// of 2^-149 at least.
__device__ __forceinline__ double ns_unit(double s, double eps) { return s == 0.0 ? 1.0 : 1.0 / (sqrt(s) + eps); }

// partial sums of a matrix: one per 64 x 64 tile of it, at most NS_PARTS
__host__ __device__ __forceinline__ int ns_parts(int m, int n)
{
    const long long t = (long long)((m + 63) / 64) * ((n + 63) / 64);
    return t < NS_PARTS ? (int)t : NS_PARTS;
}

// ---- sums of squares (64 bits: any 32-bit gradient fits), the momentum on the way
__device__ __forceinline__ void ns_norm(const NsTab &a, int id, double *red)
{
    const int mi = ns_find(a.start[NS_NORM], a.nbig, id);
    const NsMat &d = a.mat[mi];
    const int parts = ns_parts(d.m, d.n), t = id - a.start[NS_NORM][mi], b = t / parts, part = t - b * parts;
    const char *src = ns_src(a, d, b);
    const int rows = d.tall ? d.n : d.m, cols = d.tall ? d.m : d.n, tc = (cols + 63) / 64, tiles = (rows + 63) / 64 * tc;
    double s = 0.0;
    for (int k = part; k < tiles; k += parts) {
        float v[16];
        ns_load_tile(a, d, src, k / tc * 64, k % tc * 64, true, v);
#pragma unroll
        for (int q = 0; q < 16; ++q) s = fma((double)v[q], (double)v[q], s);
    }
    s = p2c_wave_sum_f64(s);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) reinterpret_cast<double *>(a.ws + d.ws + b * d.ws_bs)[part] = red[0] + red[1] + red[2] + red[3];
}

// Tiles of a symmetric product that reach the diagonal or lie above it: rows of tiles i, of tile rows `tr` high and `tb` wide, nt of them across
__host__ __device__ __forceinline__ int ns_sym_tiles(int side, int tr, int tb)
{
    const int q = tr / tb, rows = side / tr, nt = side / tb;
    return rows * nt - q * (rows * (rows - 1) / 2);
}
// tile t of them, row by row -> (i, j)
__device__ __forceinline__ void ns_triangle(int t, int nt, int q, int &i, int &j)
{
    i = 0;
    while (t >= nt - q * i) { t -= nt - q * i; ++i; }
    j = q * i + t;
}
__host__ __device__ __forceinline__ int ns_tile_rows(int tile) { return tile == 96 ? 128 : tile; }
__host__ __device__ __forceinline__ int ns_tile_cols(int tile) { return tile == 96 ? 64 : tile; }
__host__ __device__ constexpr int ns_waves(int cols) { return cols == 32 ? 1 : 4; }

// table and records, spread over a launch's threads
__device__ __forceinline__ void ns_records(const NsTab &a)
{
    if (blockIdx.x == 0)
        for (int k = threadIdx.x; k < (int)(sizeof(NsTab) / 4); k += 256) reinterpret_cast<int *>(a.ws)[k] = reinterpret_cast<const int *>(&a)[k];
    NsRec *rec = reinterpret_cast<NsRec *>(a.ws + NS_TAB_BYTES);
    for (int k = blockIdx.x * 256 + threadIdx.x; k < a.nsym + a.nall; k += gridDim.x * 256) {
        const bool sym = k < a.nsym;
        const int id = sym ? k : k - a.nsym, *start = a.start[sym ? NS_SYM : NS_ALL], tile = sym ? a.tsym : a.tall, mi = ns_find(start, a.nbig, id);
        const NsMat &d = a.mat[mi];
        const int tr = ns_tile_rows(tile), tb = ns_tile_cols(tile), mt = d.mP / tb, per = sym ? ns_sym_tiles(d.mP, tr, tb) : mt * (d.nP / tr);
        int t = ns_xcd_order(id - start[mi], start[mi + 1] - start[mi]);
        NsRec r;
        r.mi = mi; r.mP = d.mP; r.nP = d.nP;
        r.b = t / per;
        t -= r.b * per;
        if (sym) ns_triangle(t, mt, tr / tb, r.ti, r.tj);
        else { r.ti = t / mt; r.tj = t - r.ti * mt; }
        r.w = (unsigned long long)(a.ws + d.ws + r.b * d.ws_bs);
        rec[k] = r;
    }
}

// ---- X_0: a 64 x 64 tile normalised and stored as S and T
__global__ void __launch_bounds__(256) ns_begin_kernel(const NsTab a)
{
    __shared__ float x[64][65];
    __shared__ double red[4];
    const int id = blockIdx.x, mi = ns_find(a.start[NS_TILES], a.nbig, id);
    const NsMat &d = a.mat[mi];
    const int rows = d.tall ? d.nP : d.mP, cols = d.tall ? d.mP : d.nP, tc = cols / 64, per = rows / 64 * tc;
    const int t = id - a.start[NS_TILES][mi], b = t / per, tt = t - b * per, r0 = tt / tc * 64, c0 = tt % tc * 64, tid = threadIdx.x;
    char *w = a.ws + d.ws + b * d.ws_bs;
    float v[16];
    ns_load_tile(a, d, ns_src(a, d, b), r0, c0, false, v);
    ns_records(a);
    const int parts = ns_parts(d.m, d.n);
    double s = 0.0;
    for (int k = tid; k < parts; k += 256) s += reinterpret_cast<const double *>(w)[k];
    s = p2c_wave_sum_f64(s);
    if ((tid & 63) == 0) red[tid >> 6] = s;
    __syncthreads();
    const double inv = (double)NS_SCALE * ns_unit(red[0] + red[1] + red[2] + red[3], a.eps);
#pragma unroll
    for (int q = 0; q < 16; ++q) x[(tid >> 6) + 4 * q][tid & 63] = (float)((double)v[q] * inv);
    __syncthreads();
    // the image whose rows are the matrix' rows, and the other
    char *R = d.tall ? ns_T(w, d, 0) : ns_S(w), *C = d.tall ? ns_S(w) : ns_T(w, d, 0);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int e = tid + 256 * q, r = e >> 3, c8 = (e & 7) * 8;
        float u[8];
        h16x8 hi, lo;
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = x[r][c8 + k];
        ns_split8(u, hi, lo);
        h16x8 *o = reinterpret_cast<h16x8 *>(R + ((size_t)((c0 + c8) >> 5) * rows + r0 + r) * 128 + (c8 & 31) * 4);
        o[0] = hi; o[1] = lo;
#pragma unroll
        for (int k = 0; k < 8; ++k) u[k] = x[c8 + k][r];
        ns_split8(u, hi, lo);
        o = reinterpret_cast<h16x8 *>(C + ((size_t)((r0 + c8) >> 5) * cols + c0 + r) * 128 + (c8 & 31) * 4);
        o[0] = hi; o[1] = lo;
    }
}

// four values of a lane times a power of two as two fp16 each
__device__ __forceinline__ void ns_split4(float v0, float v1, float v2, float v3, float f, h16x4 &hi, h16x4 &lo)
{
    const float v[4] = {v0, v1, v2, v3};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        hi[e] = (_Float16)(v[e] * f);
        lo[e] = (_Float16)__builtin_fmaf(v[e], f, -(float)hi[e]);
    }
}

// 4 x 4 half words across a quad of lanes: in, word e of lane q is M[e][q]; out, lane q holds M[q][0..3]
__device__ __forceinline__ uint2 ns_quad_transpose(uint2 r, int lane)
{
    const uint32_t sel = lane & 1 ? 0x03020706u : 0x05040100u;             // odd: {high of the partner, own high}; even: {own low, low of the partner}
    const uint32_t a0 = __builtin_amdgcn_perm((uint32_t)p2c_dpp<0xB1>((int)r.x), r.x, sel), a1 = __builtin_amdgcn_perm((uint32_t)p2c_dpp<0xB1>((int)r.y), r.y, sel);
    const bool up = (lane & 2) != 0;
    const uint32_t y = (uint32_t)p2c_dpp<0x4E>((int)(up ? a0 : a1));
    return up ? make_uint2(y, a1) : make_uint2(a0, y);
}

// ---- one product of a step for every matrix.  PH 1: A = S S^T.  2: B = b A + c A A^T.  3: T' = a T + T B^T (and S').  4: as 3, into the result.
// Tile TR x TB: 128 x 128 or 128 x 64 (four waves of 64 x 64 or 64 x 32), 64 x 64 (four of 32 x 32) or 32 x 32 (one), for each of KG groups that share
// the k range (group g takes blocks g, g + KG, ...).  NST stages of one block (32 k, 128 bytes a row) are filled by direct copies, NST - 1 of them in flight.
// A block is multiplied in two halves; the fragments of the next half are read, and the copies issued, BETWEEN the products of this one: instructions issue
// in order, and copies in one go kept a wave from its products until the memory pipe had taken them (copies and products took the sum of their times;
// 8 x 1024 x 2048: T' 136 us with reads, copies and products in turn, 123 with the reads a half ahead, 112 with the copies spread).
// The addend b A, a T is the product's own first operand, so it is picked up when its block passes by: a product with the unit matrix, exact, into sums of
// its own (into the product's it would be rounded again by every later step).  Fetched from memory in the results' layout it cost 10000 clocks a tile.
// What bounds it at 8 x 1024 x 2048: T' runs 103 GFLOP in 107 us (960 TFLOP/s; a large library product, under the same power limit, 1160 - 1220).  Power sets the clock
// (1.75 GHz; the same launches on zeros take 24 us less); the rest of the distance has not been attributed.  A: 73 us for 576 tiles on 512 places, a second round for 64.
template <int TR, int TB, int KG, int NST, int PH>
__global__ void __launch_bounds__(64 * ns_waves(TB) * KG, 2) ns_product_kernel(const NsTab *__restrict__ tab, const NsRec *__restrict__ recs, const float ca, const float cb, const int cur)
{
    constexpr int WG = ns_waves(TB), RB = 128, TILE = (TR + TB) * RB, STAGE = KG * TILE, NX = TR >= 128 ? 2 : 1, NY = TB / 64 < 1 ? 1 : TB / 64, LPW = TILE / 1024 / WG;
    constexpr int GP = 4 / KG;                      // row groups of a piece (8 g + 4 h + 0..3) that a k-group finishes
    static_assert(KG == 1 || NX * NY == 1, "");
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const NsRec d = recs[blockIdx.x];
    const int tid = threadIdx.x, lane = tid & 63, gw = __builtin_amdgcn_readfirstlane(tid >> 6), wave = gw % WG, kg = gw / WG, il = lane & 31, h = lane >> 5;
    const int ti = d.ti, tj = d.tj;                 // tile rows of P and of Q
    char *w = reinterpret_cast<char *>(d.w);
    const char *P, *Q;
    int K;
    if (PH == 1) { P = Q = ns_S(w); K = d.nP; }
    else if (PH == 2) { P = Q = ns_A(w, d); K = d.mP; }
    else { P = ns_T(w, d, cur); Q = ns_B(w, d); K = d.mP; }
    const long long pb = (long long)(PH <= 2 ? d.mP : d.nP) * RB, qb = (long long)d.mP * RB;       // bytes of a block of 32 k
    P += ti * TR * RB;
    Q += tj * TB * RB;
    const int KB = K / 32, IT = (KB + KG - 1) / KG;
    const int wr = WG == 1 ? 0 : (wave >> 1) * (32 * NX), wc = WG == 1 ? 0 : (wave & 1) * (32 * NY);

    f32x16 acc[NX][NY], own[NX][NY];
#pragma unroll
    for (int p = 0; p < NX; ++p)
#pragma unroll
        for (int q = 0; q < NY; ++q)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[p][q][r] = own[p][q][r] = 0.f;
    // a block's rows are one run of memory, so a wave's copies are 1 KB pieces of it: a scalar base and one lane offset (odd pieces of a single wave: the other swizzle)
    const unsigned lo = lane / 8 * RB + (((lane & 7) ^ p2c_tile_swz<RB>(wave * 8 + lane / 8)) << 4);
    auto copy = [&](int it, int stage, int i) {     // piece i of this wave (past the end: the last block again, into a stage that is not multiplied: the count in flight stays exact)
        constexpr int NP = TR * RB / 1024 / WG;
        const int k = min(it * KG + kg, KB - 1), at = (wave + (i < NP ? i : i - NP) * WG) * 1024;
        char *st = smem + stage * STAGE + kg * TILE + (i < NP ? 0 : TR * RB) + at;
        const char *src = (i < NP ? P + k * pb : Q + k * qb) + at;
        p2c_tile_piece(src + (WG == 1 && (i & 1) ? lo ^ 64 : lo), st);
    };
    struct Frags { h16x8 p[NX][2], q[NY][2]; };
    constexpr int M = 3 * NX * NY, R = 2 * (NX + NY);
    auto read = [&](Frags &f, int stage, int half, int i) {                  // fragment i of R
        const char *ps = smem + stage * STAGE + kg * TILE, *qs = ps + TR * RB;
        const int pl = i / (NX + NY), x = i % (NX + NY), y = x - NX, c = 4 * half + 2 * h + pl;
        if (x < NX) f.p[x][pl] = *reinterpret_cast<const h16x8 *>(ps + p2c_tile_at<RB>(wr + x * 32 + il, c));
        else f.q[y][pl] = *reinterpret_cast<const h16x8 *>(qs + p2c_tile_at<RB>(wc + y * 32 + il, c));
    };
    // the reads of the next half go between the products of this one, two for each of the first; so do the copies, evenly
    auto reads = [&](Frags &f, int stage, int half, int n) {
#pragma unroll
        for (int i = 2 * n; i < (n + 1 == M ? R : 2 * n + 2) && i < R; ++i) read(f, stage, half, i);
    };
    const int cy = (tj * TB + wc) >> 5;             // the k-tile of this wave's first 32 columns
    // after product n: then(n)
    auto multiply = [&](const Frags &f, int it, int half, auto then) {
        const bool on = KG == 1 || it * KG + kg < KB;
        const int k = it * KG + kg;
#pragma unroll
        for (int pr = 0; pr < 3; ++pr)              // small products first
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int y = 0; y < NY; ++y) {
                    if (on) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.p[x][pr == 1], f.q[y][pr == 0], acc[x][y], 0, 0, 0);
                    then((pr * NX + x) * NY + y);
                }
        if (!on) return;
        if (PH != 1) {
#pragma unroll
            for (int y = 0; y < NY; ++y)
                if (k == cy + y) {
                    h16x8 one;                      // the unit matrix' half of this step as a fragment
#pragma unroll
                    for (int e = 0; e < 8; ++e) one[e] = (_Float16)(16 * half + 8 * h + e == il ? 1.f : 0.f);
#pragma unroll
                    for (int x = 0; x < NX; ++x)
#pragma unroll
                        for (int pl = 1; pl >= 0; --pl) own[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.p[x][pl], one, own[x][y], 0, 0, 0);
                }
        }
    };
#pragma unroll
    for (int it = 0; it < NST; ++it)
#pragma unroll
        for (int i = 0; i < LPW; ++i) copy(it, it, i);
    Frags f0, f1;
    int now = 0;                                    // stage of block it
    p2c_tile_wait<(NST - 1) * LPW>();
#pragma unroll
    for (int i = 0; i < R; ++i) read(f0, 0, 0, i);
    for (int it = 0; it < IT; ++it) {
        const int next = now + 1 == NST ? 0 : now + 1;
        __builtin_amdgcn_s_waitcnt(15 | 7 << 4 | 3 << 14);          // f0 has arrived (lgkmcnt 0): known before the next reads are issued, or the products would wait for those
        multiply(f0, it, 0, [&](int n) {
            reads(f1, now, 1, n);
            asm volatile("" ::: "memory");          // (read here, not where they are used)
            __builtin_amdgcn_sched_barrier(0);
        });
        p2c_tile_wait<(NST - 2) * LPW>();           // block it + 1 is here; everybody has read block it
        // issued in one go, the copies held up the wave and its products with it: 123 us instead of 112 for a T' of 8 x 1024 x 2048
        multiply(f1, it, 1, [&](int n) {
            reads(f0, next, 0, n);
#pragma unroll
            for (int i = n * LPW / M; i < (n + 1) * LPW / M; ++i) copy(it + NST, now, i);
            asm volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        });
        now = next;
    }
    p2c_tile_wait<0>();                             // the surplus copies have landed: the stages are free

    // ---- epilogue.  A lane holds column il of a 32 x 32 piece, rows 8 g + 4 h + (0..3): four consecutive k of the transposed image as they are, of the straight one
    // after a 4 x 4 exchange in the lane's quad.  Both images of a piece are put together in LDS and leave as whole 128-byte lines.
    const bool mirror = PH == 3 || (PH <= 2 && tj * TB >= (ti + 1) * TR);       // (the tiles over the diagonal cover both sides of it)
    char *o1 = PH == 1 ? ns_A(w, d) : PH == 2 ? ns_B(w, d) : ns_T(w, d, cur ^ 1);
    char *o2 = PH == 3 ? ns_S(w) : o1;
    const int rows1 = PH <= 2 ? d.mP : d.nP;
    constexpr int LDF = 33;                         // floats of a staged row of the result
    char *piece = smem + (KG == 1 ? 0 : KG * WG * 4 * 64 * 16) + wave * 8192;
    auto finish = [&](int g, const float (&c)[4]) { // c: the new values (scaled), or the result
        if (PH == 4) {
#pragma unroll
            for (int e = 0; e < 4; ++e) reinterpret_cast<float *>(piece)[(8 * g + 4 * h + e) * LDF + il] = c[e];
        } else {
            h16x4 hi, lo;
            ns_split4(c[0], c[1], c[2], c[3], 1.0f, hi, lo);
            const int at = p2c_tile_at<128>(il, 2 * g) + 8 * h;
            *reinterpret_cast<h16x4 *>(piece + 4096 + at) = hi;
            *reinterpret_cast<h16x4 *>(piece + 4096 + (at ^ 16)) = lo;
            const uint2 th = ns_quad_transpose(__builtin_bit_cast(uint2, hi), lane), tl = ns_quad_transpose(__builtin_bit_cast(uint2, lo), lane);
            const int at1 = p2c_tile_at<128>(8 * g + 4 * h + (lane & 3), (il >> 3) * 2) + (il & 4) * 2;
            *reinterpret_cast<uint2 *>(piece + at1) = th;
            *reinterpret_cast<uint2 *>(piece + (at1 ^ 16)) = tl;
        }
    };
    // out: `first` of `count` lanes that share a piece; r0, c0: its place
    auto leave = [&](int r0, int c0, int first, int count) {
        if (PH == 4) {
            const NsMat &m = tab->mat[d.mi];
            const float *stage = reinterpret_cast<const float *>(piece);
            for (int e0 = first; e0 < 1024; e0 += 4 * count) {                      // lanes run along the contiguous side of the output
                float o[4];
                auto i = [&](int q) { const int e = e0 + q * count; return m.tall ? e & 31 : e >> 5; };
                auto j = [&](int q) { const int e = e0 + q * count; return m.tall ? e >> 5 : e & 31; };
#pragma unroll
                for (int q = 0; q < 4; ++q) o[q] = stage[j(q) * LDF + i(q)] * NS_INV;
                ns_store_n(*tab, m, d.b, o, [&](int q) { return c0 + i(q); }, [&](int q) { return r0 + j(q); });
            }
        } else {
#pragma unroll
            for (int u = first; u < 256; u += count) {
                const int r = u >> 3, p = u & 7, c = p ^ p2c_tile_swz<128>(r);
                *reinterpret_cast<f32x4 *>(o1 + ((size_t)(c0 >> 5) * rows1 + r0 + r) * 128 + c * 16) = *reinterpret_cast<const f32x4 *>(piece + u * 16);
                if (mirror) *reinterpret_cast<f32x4 *>(o2 + ((size_t)(r0 >> 5) * d.mP + c0 + r) * 128 + c * 16) = *reinterpret_cast<const f32x4 *>(piece + 4096 + u * 16);
            }
        }
    };
    if (KG == 1) {
#pragma unroll
        for (int x = 0; x < NX; ++x)
#pragma unroll
            for (int y = 0; y < NY; ++y) {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    float c[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        c[e] = PH == 1 ? acc[x][y][4 * g + e] * NS_INV : __builtin_fmaf(ca, own[x][y][4 * g + e], cb * (acc[x][y][4 * g + e] * NS_INV));
                    finish(g, c);
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                leave(ti * TR + wr + x * 32, tj * TB + wc + y * 32, lane, 64);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
    } else {
        // the groups' sums meet in LDS; group k finishes the row groups GP k ... GP k + GP - 1 of its wave's piece
        f32x4 *sums = reinterpret_cast<f32x4 *>(smem);                               // [group][wave][g][lane]
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            f32x4 c;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                c[e] = PH == 1 ? acc[0][0][4 * g + e] * NS_INV : __builtin_fmaf(ca, own[0][0][4 * g + e], cb * (acc[0][0][4 * g + e] * NS_INV));
            sums[((kg * WG + wave) * 4 + g) * 64 + lane] = c;
        }
        __syncthreads();
#pragma unroll
        for (int g = 0; g < GP; ++g) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KG; ++k) {
                const f32x4 v = sums[((k * WG + wave) * 4 + kg * GP + g) * 64 + lane];
#pragma unroll
                for (int e = 0; e < 4; ++e) c[e] += v[e];
            }
            finish(kg * GP + g, c);
        }
        __syncthreads();
        leave(ti * TR + wr, tj * TB + wc, kg * 64 + lane, 64 * KG);
    }
}

struct NsCoef { int steps; float c[16][3]; };

// 8 elements from offset `at` on, `cs` apart, of which `left` exist (zeros for the others): in 16-byte pieces where they are whole and neighbours
typedef f32x4 f32x4_u __attribute__((aligned(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef u16x8 u16x8_u __attribute__((aligned(2)));
__device__ __forceinline__ float ns_wide(uint16_t u, int dtype) { return dtype == 1 ? __uint_as_float((uint32_t)u << 16) : (float)__builtin_bit_cast(_Float16, u); }
__device__ __forceinline__ uint16_t ns_narrow(float v, int dtype) { return dtype == 1 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v); }
__device__ __forceinline__ void ns_get8(const char *p, long long at, long long cs, int left, int dtype, float (&v)[8])
{
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = 0.f;
    if (left >= 8 && cs == 1) {
        if (dtype == 0) {
            const f32x4_u *q = reinterpret_cast<const f32x4_u *>(p + at * 4);
            const f32x4 x = q[0], y = q[1];
#pragma unroll
            for (int k = 0; k < 4; ++k) { v[k] = x[k]; v[4 + k] = y[k]; }
        } else {
            const u16x8 x = *reinterpret_cast<const u16x8_u *>(p + at * 2);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = ns_wide(x[k], dtype);
        }
    } else {
#pragma unroll 1
        for (int k = 0; k < 8; ++k)
            if (k < left) {
                const float x = dtype == 0 ? *reinterpret_cast<const float *>(p + (at + k * cs) * 4) : ns_wide(*reinterpret_cast<const uint16_t *>(p + (at + k * cs) * 2), dtype);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = e == k ? x : v[e];
            }
    }
}
__device__ __forceinline__ void ns_put8(char *p, long long at, long long cs, int left, int dtype, const float (&v)[8])
{
    if (left >= 8 && cs == 1) {
        if (dtype == 0) {
            f32x4_u *q = reinterpret_cast<f32x4_u *>(p + at * 4);
            q[0] = f32x4{v[0], v[1], v[2], v[3]};
            q[1] = f32x4{v[4], v[5], v[6], v[7]};
        } else {
            u16x8 x;
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] = ns_narrow(v[k], dtype);
            *reinterpret_cast<u16x8_u *>(p + at * 2) = x;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < left) {
                if (dtype == 0) *reinterpret_cast<float *>(p + (at + k * cs) * 4) = v[k];
                else *reinterpret_cast<uint16_t *>(p + (at + k * cs) * 2) = ns_narrow(v[k], dtype);
            }
    }
}

// ---- matrices of up to 16384 elements (sides padded to 64: 128 x 128, 64 x 256): one workgroup each, all steps without leaving LDS.  The tiled form is
// a chain of 17 launches of 4 us.  Here a call of 128 x 128 is 52 us (64 tiled): fifteen products of 3.4.  A product's matrix instructions and its operand reads
// out of LDS (384 KB) take 1.3 - 1.5 us each and overlap; the rest lies between the products: six workgroup barriers a step, as S, then A, then B share one region
// (S is read by the first product only, and a X comes from the registers, which hold X in 32 bits in the layout of the products' results), the splitting and storing of
// every result, and A, which is read back for b A.
constexpr int NS_MID = 16384;

struct NsMidImage { int base, rows; };                          // offset in LDS; [k-tile][row][128 bytes], chunks permuted as in tile_dma.h

// offset of the hi chunk of 8 k; the lo chunk is 16 bytes apart before the permutation (chunk c and c ^ 1): its offset is this one ^ 16
__device__ __forceinline__ int ns_mid_at(const NsMidImage &m, int row, int k) { return m.base + (k >> 5) * (m.rows * 128) + p2c_tile_at<128>(row, (k & 31) >> 3 << 1); }

// 16 values of a lane (rows 8 g + 4 h + 0..3 of a 32 x 32 piece, times a power of two) as 4 x 4 consecutive k of image row `row`, k-tile k0 / 32
__device__ __forceinline__ void ns_mid_put(char *lds, const NsMidImage &m, int row, int k0, int h, const f32x16 &v, float f)
{
    const int at = ns_mid_at(m, row, k0) + 8 * h;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        h16x4 hi, lo;
        ns_split4(v[4 * g], v[4 * g + 1], v[4 * g + 2], v[4 * g + 3], f, hi, lo);
        *reinterpret_cast<h16x4 *>(lds + (at ^ (32 * g))) = hi;
        *reinterpret_cast<h16x4 *>(lds + (at ^ (32 * g + 16))) = lo;
    }
}

__global__ void __launch_bounds__(512) ns_mid_kernel(const NsTab a, const NsCoef co)
{
    extern __shared__ __attribute__((aligned(1024))) char smem[];
    const int mi = ns_find(a.start[NS_ALL], a.nbig, blockIdx.x);
    const NsMat &d = a.mat[mi];
    const int b = blockIdx.x - a.start[NS_ALL][mi], tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), il = lane & 31, h = lane >> 5;
    const int mt = d.mP >> 5, nt = d.nP >> 5, xb = d.mP * d.nP * 4;
    const NsMidImage S = {0, d.mP}, T = {xb, d.nP};               // A and B are images of mP rows in S's place
    double *red = reinterpret_cast<double *>(smem + 2 * xb);

    // ---- the matrix: 8 consecutive columns of a row per unit, at most 4 units a thread
    const int rows = d.tall ? d.n : d.m, cols = d.tall ? d.m : d.n, c8n = (d.tall ? d.mP : d.nP) >> 3, units = (d.tall ? d.nP : d.mP) * c8n;
    const char *src = ns_src(a, d, b);
    const float rc8 = 1.0f / c8n;
    int ur[4], uc[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int u = tid + 512 * q;
        ur[q] = (int)((u + 0.5f) * rc8);                        // u / c8n (u < 2048)
        uc[q] = (u - ur[q] * c8n) * 8;
    }
    float v[4][8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int left = tid + 512 * q < units && ur[q] < rows ? cols - uc[q] : 0;
        ns_get8(src, ur[q] * d.src_rs + uc[q] * d.src_cs, d.src_cs, left, a.dtype, v[q]);
    }
    if (a.muon) {
        float m[4][8];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int left = tid + 512 * q < units && ur[q] < rows ? cols - uc[q] : 0;
            ns_get8((const char *)d.mom, (long long)ur[q] * cols + uc[q], 1, left, 0, m[q]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int left = tid + 512 * q < units && ur[q] < rows ? cols - uc[q] : 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                m[q][k] = __builtin_fmaf(a.mu, m[q][k], (1.0f - a.mu) * v[q][k]);
                v[q][k] = a.muon == 2 ? __builtin_fmaf(a.mu, m[q][k], (1.0f - a.mu) * v[q][k]) : m[q][k];
            }
            ns_put8((char *)d.mom, (long long)ur[q] * cols + uc[q], 1, left, 0, m[q]);
        }
    }
    double s = 0.0;
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int k = 0; k < 8; ++k) s = fma((double)v[q][k], (double)v[q][k], s);
    s = p2c_wave_sum_f64(s);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += red[k];
    const double inv = (double)NS_SCALE * ns_unit(s, a.eps);
    const float finv = (float)inv;
    if (finv > 1e-30f && finv < 1e30f) {                        // the factor of ordinary magnitudes is a 32-bit number
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int k = 0; k < 8; ++k) v[q][k] *= finv;
    } else {
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {                           // (in two factors, each in range)
            const double half = e ? inv / (double)(float)sqrt(inv) : (double)(float)sqrt(inv);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int k = 0; k < 8; ++k) v[q][k] = (float)((double)v[q][k] * half);
        }
    }
    const NsMidImage &R = d.tall ? T : S, &C = d.tall ? S : T;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (tid + 512 * q < units) {
            float w[8];
            h16x8 hi, lo;
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = v[q][k];
            ns_split8(w, hi, lo);
            const int at = ns_mid_at(R, ur[q], uc[q]);
            *reinterpret_cast<h16x8 *>(smem + at) = hi;
            *reinterpret_cast<h16x8 *>(smem + (at ^ 16)) = lo;
        }
    __syncthreads();

    // fragments: row block `rb` of an image at k-step ks (16 k), plane pl
    auto frag = [&](const NsMidImage &m, int rb, int ks, int pl) {
        return *reinterpret_cast<const h16x8 *>(smem + (ns_mid_at(m, rb * 32 + il, ks * 16 + 8 * h) ^ (16 * pl)));
    };
    h16x8 one[2];                                               // the unit matrix of one k-tile as a fragment: a product with it re-lays a matrix exactly
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) one[t][e] = (_Float16)(16 * t + 8 * h + e == il ? 1.f : 0.f);
    auto clear = [&](f32x16 &c) {
#pragma unroll
        for (int r = 0; r < 16; ++r) c[r] = 0.f;
    };
    // C[row block rb][column block cb] of an image itself: lane = column, rows in the registers
    auto self = [&](const NsMidImage &m, int rb, int cb, f32x16 &c) {
        clear(c);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int pl = 1; pl >= 0; --pl) c = __builtin_amdgcn_mfma_f32_32x32x16_f16(frag(m, rb, 2 * cb + t, pl), one[t], c, 0, 0, 0);
    };
    f32x16 acc[2], x[2];
    // the other image
    const int rbn = R.rows >> 5, pairs = C.rows >> 6;           // at most 8 units of 32 rows x 64 columns: one a wave, here and in every product
    if (wave < rbn * pairs) {
        const int rb = wave / pairs, cb = wave % pairs * 2;
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            self(R, rb, cb + y, acc[y]);
            ns_mid_put(smem, C, (cb + y) * 32 + il, rb * 32, h, acc[y], 1.0f);
        }
    }
    const int mp = mt >> 1, r3 = wave / mp, c3 = wave % mp * 2;  // this wave's unit: of the m x m products where it is one, of T'
    const bool in_sym = wave < mt * mp, in_all = wave < nt * mp;
    if (in_all) {                                               // X in the layout of T': lane = i, j in the registers; from the image that is there
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            if (d.tall) {
                self(T, r3, c3 + y, x[y]);
            } else {
                clear(x[y]);
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int pl = 1; pl >= 0; --pl) x[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(one[t], frag(S, c3 + y, 2 * r3 + t, pl), x[y], 0, 0, 0);
            }
        }
    }
    __syncthreads();
    // A k-tile's fragments (chunk 2 (2 s + h) + pl of a row: s and pl are bits 6 and 4 of its offset, whatever the permutation) are read while the one
    // before is multiplied: read and multiplied in turn, a product took 6100 clocks for 3100 of either.
    struct Frags { h16x8 p[2][2], q[2][2][2]; };
    auto product = [&](const NsMidImage &p, const NsMidImage &q, int KT) {
        clear(acc[0]);
        clear(acc[1]);
        int op = ns_mid_at(p, r3 * 32 + il, 8 * h), oq[2] = {ns_mid_at(q, c3 * 32 + il, 8 * h), ns_mid_at(q, c3 * 32 + 32 + il, 8 * h)};
        const int sp = p.rows * 128, sq = q.rows * 128;
        auto read = [&](Frags &f) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int pl = 0; pl < 2; ++pl) {
                    f.p[t][pl] = *reinterpret_cast<const h16x8 *>(smem + (op ^ (64 * t + 16 * pl)));
#pragma unroll
                    for (int y = 0; y < 2; ++y) f.q[t][y][pl] = *reinterpret_cast<const h16x8 *>(smem + (oq[y] ^ (64 * t + 16 * pl)));
                }
            op += sp;
            oq[0] += sq;
            oq[1] += sq;
        };
        auto multiply = [&](const Frags &f) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int pr = 0; pr < 3; ++pr)
#pragma unroll
                    for (int y = 0; y < 2; ++y) acc[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.p[t][pr == 1], f.q[t][y][pr == 0], acc[y], 0, 0, 0);
        };
        Frags f0, f1;
        read(f0);
        for (int kt = 0; kt < KT; kt += 2) {                    // (KT is even: the sides are multiples of 64)
            read(f1);
            __builtin_amdgcn_sched_barrier(0);
            multiply(f0);
            __builtin_amdgcn_sched_barrier(0);
            if (kt + 2 < KT) read(f0);
            __builtin_amdgcn_sched_barrier(0);
            multiply(f1);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int st = 0; st < co.steps; ++st) {
        const float c0 = co.c[st][0], c1 = co.c[st][1], c2 = co.c[st][2];
        asm volatile("" ::"s"(c0), "s"(c1), "s"(c2));           // here now: a scalar load in flight would make every wait below a wait for all of LDS
        if (in_sym) product(S, S, nt);
        __syncthreads();
        if (in_sym) {                                           // (A is symmetric: its transposed image is its image)
#pragma unroll
            for (int y = 0; y < 2; ++y) ns_mid_put(smem, S, (c3 + y) * 32 + il, r3 * 32, h, acc[y], NS_INV);
        }
        __syncthreads();
        if (in_sym) {
            product(S, S, mt);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int at = ns_mid_at(S, (c3 + y) * 32 + il, r3 * 32) + 8 * h;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const h16x4 oh = *reinterpret_cast<const h16x4 *>(smem + (at ^ (32 * g))), ol = *reinterpret_cast<const h16x4 *>(smem + (at ^ (32 * g + 16)));
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[y][4 * g + e] = __builtin_fmaf(c1, (float)oh[e] + (float)ol[e], (c2 * NS_INV) * acc[y][4 * g + e]);
                }
            }
        }
        __syncthreads();
        if (in_sym) {
#pragma unroll
            for (int y = 0; y < 2; ++y) ns_mid_put(smem, S, (c3 + y) * 32 + il, r3 * 32, h, acc[y], 1.0f);
        }
        __syncthreads();
        if (in_all) {
            product(T, S, mt);
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int r = 0; r < 16; ++r) x[y][r] = __builtin_fmaf(c0, x[y][r], acc[y][r] * NS_INV);
        }
        if (st + 1 == co.steps) break;
        __syncthreads();
        if (in_all) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int i = (c3 + y) * 32 + il, at = ns_mid_at(S, i, r3 * 32) + 8 * h;
                // T': rows r3 32 + 8 g + 4 h + (lane & 3), columns of the lane's quad; 8 rows on, the permutation's bits 4-6 change by (8 / 2) << 4
                const int i4 = i & ~3, at_t = ns_mid_at(T, r3 * 32 + 4 * h + (lane & 3), i4) + (i4 & 4) * 2;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    h16x4 hi, lo;
                    ns_split4(x[y][4 * g], x[y][4 * g + 1], x[y][4 * g + 2], x[y][4 * g + 3], 1.0f, hi, lo);
                    *reinterpret_cast<h16x4 *>(smem + (at ^ (32 * g))) = hi;
                    *reinterpret_cast<h16x4 *>(smem + (at ^ (32 * g + 16))) = lo;
                    const uint2 th = ns_quad_transpose(__builtin_bit_cast(uint2, hi), lane), tl = ns_quad_transpose(__builtin_bit_cast(uint2, lo), lane);
                    const int t = (at_t + g * 1024) ^ ((g & 1) * 64);
                    *reinterpret_cast<uint2 *>(smem + t) = th;
                    *reinterpret_cast<uint2 *>(smem + (t ^ 16)) = tl;
                }
            }
        }
        __syncthreads();
    }
    // the result through LDS (the images are done with), out 8 columns of a row at a time
    __syncthreads();
    float *stage = reinterpret_cast<float *>(smem);
    const int lds = (d.tall ? d.mP : d.nP) + 4;                 // (16384 + 4 x 256 floats at most: within the two images)
    if (in_all) {
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int i = (c3 + y) * 32 + il, j = r3 * 32 + 8 * g + 4 * h;
                if (d.tall) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) stage[(j + e) * lds + i] = x[y][4 * g + e];
                } else {
                    *reinterpret_cast<f32x4 *>(stage + i * lds + j) = f32x4{x[y][4 * g], x[y][4 * g + 1], x[y][4 * g + 2], x[y][4 * g + 3]};
                }
            }
    }
    __syncthreads();
    char *dst = d.dst + b * d.dst_bs * (a.dtype == 0 ? 4 : 2);
    float o[4][8];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int left = tid + 512 * q < units && ur[q] < rows ? cols - uc[q] : 0;
        if (a.muon) ns_get8(dst, ur[q] * d.dst_rs + uc[q] * d.dst_cs, d.dst_cs, left, 0, o[q]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int left = tid + 512 * q < units && ur[q] < rows ? cols - uc[q] : 0;
        if (left > 0) {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(stage + ur[q] * lds + uc[q]), hi = *reinterpret_cast<const f32x4 *>(stage + ur[q] * lds + uc[q] + 4);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float r = (k < 4 ? lo[k & 3] : hi[k & 3]) * NS_INV;
                o[q][k] = a.muon ? o[q][k] * d.decay - d.scale * r : r;
            }
            ns_put8(dst, ur[q] * d.dst_rs + uc[q] * d.dst_cs, d.dst_cs, left, a.dtype, o[q]);
        }
    }
}

// ---- small side <= 16: one workgroup per matrix, in the m x m space and in 64 bits.  X_k = Q_k X_0 with Q and A polynomials of A_0 = X_0 X_0^T:
// q = a + bA + cA^2, Q <- q Q, A <- q A q.  G is read twice and nothing else moves.  64 bits are what this form needs (A holds SQUARED singular
// values and a rounding grows by a^2 per step: 2.5e5 over five); at this size they cost less than the launches of the tiled form.
constexpr int NS_XS = 2064;                                     // floats of a chunk of X: m rows of 128 ... 512 elements, each padded by one

struct NsSmallLds {
    double A[NS_SMALL][NS_SMALL + 1], Q[NS_SMALL][NS_SMALL + 1], U[NS_SMALL][NS_SMALL + 1], V[NS_SMALL][NS_SMALL + 1];
    double part[4][256];
    float x[NS_XS];
};

template <int M>
__device__ __forceinline__ double ns_dot(const double (*x)[NS_SMALL + 1], const double (*y)[NS_SMALL + 1], int i, int j)
{
    double s = 0.0;
#pragma unroll 8
    for (int k = 0; k < M; ++k) s = fma(x[i][k], y[k][j], s);
    return s;
}

// M: a power of two >= m, at least 4; the matrices are padded with zeros to M.  The 2 x 2 blocks of the M x M Gram matrix take (M/2)^2 threads; the
// others share the long side.
template <int M>
__device__ __forceinline__ void ns_small(const NsTab &a, const NsCoef &co, int mi, int b, NsSmallLds &l)
{
    constexpr int BL = M / 2, SPLIT = 256 / (BL * BL), JC = 2048 / M, LDX = JC + 1;
    static_assert(M <= NS_SMALL && M * LDX <= NS_XS && SPLIT <= JC, "");
    const NsMat &d = a.mat[mi];
    const int tid = threadIdx.x, m = d.m, n = d.n;
    const int blk = tid % (BL * BL), sp = tid / (BL * BL), pi = blk / BL, pj = blk % BL;
    const char *src = ns_src(a, d, b);
    double g[2][2] = {{0.0, 0.0}, {0.0, 0.0}};
    float nx[8];                                                // the next chunk, in flight under the sums of this one: 2048 elements
    auto place_of = [&](int e, int &i, int &j) {                // wide: j runs along the lanes, tall: i does
        if (d.tall) { i = e % M; j = e / M; } else { i = e / JC; j = e % JC; }
    };
    auto fetch = [&](int j0, bool first) {
        auto ii = [&](int q) { int i, j; place_of(tid + 256 * q, i, j); return i; };
        auto jj = [&](int q) { int i, j; place_of(tid + 256 * q, i, j); return j0 + j; };
        auto ok = [&](int q) { return ii(q) < m && jj(q) < n; };
        auto row = [&](int q) { return d.tall ? min(jj(q), n - 1) : min(ii(q), m - 1); };
        auto col = [&](int q) { return d.tall ? min(ii(q), m - 1) : min(jj(q), n - 1); };
        ns_load_n(src, a.dtype, nx, [&](int q) { return row(q) * d.src_rs + col(q) * d.src_cs; });
        if (a.muon) ns_momentum_n(a, d.mom, nx, first, [&](int q) { return (long long)row(q) * (d.tall ? m : n) + col(q); }, ok);
#pragma unroll
        for (int q = 0; q < 8; ++q) nx[q] = ok(q) ? nx[q] : 0.f;
    };
    auto place = [&]() {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            int i, j;
            place_of(tid + 256 * q, i, j);
            l.x[i * LDX + j] = nx[q];
        }
    };
    fetch(0, true);
    for (int j0 = 0; j0 < n; j0 += JC) {
        __syncthreads();
        place();
        __syncthreads();
        if (j0 + JC < n) fetch(j0 + JC, true);
#pragma unroll 8
        for (int j = sp; j < JC; j += SPLIT) {
            const double u0 = l.x[2 * pi * LDX + j], u1 = l.x[(2 * pi + 1) * LDX + j], v0 = l.x[2 * pj * LDX + j], v1 = l.x[(2 * pj + 1) * LDX + j];
            g[0][0] = fma(u0, v0, g[0][0]);
            g[0][1] = fma(u0, v1, g[0][1]);
            g[1][0] = fma(u1, v0, g[1][0]);
            g[1][1] = fma(u1, v1, g[1][1]);
        }
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) l.part[p][tid] = g[p >> 1][p & 1];
    __syncthreads();
    const bool on = tid < M * M;                                // an element of the M x M matrices each
    const int ei = tid / M, ej = tid % M;
    if (on) {
        const int p = (ei & 1) * 2 + (ej & 1), at = (ei >> 1) * BL + (ej >> 1);
        double s = 0.0;
#pragma unroll 8
        for (int k = 0; k < SPLIT; ++k) s += l.part[p][k * BL * BL + at];
        l.A[ei][ej] = s;
    }
    __syncthreads();
    double tr = 0.0;
#pragma unroll
    for (int k = 0; k < M; ++k) tr += l.A[k][k];
    const double inv = ns_unit(tr, a.eps);
    __syncthreads();
    if (on) {
        l.A[ei][ej] *= inv * inv;
        l.Q[ei][ej] = ei == ej ? inv : 0.0;                     // the normalisation of X_0 rides in Q
    }
    __syncthreads();
    for (int s = 0; s < co.steps; ++s) {
        const double c0 = co.c[s][0], c1 = co.c[s][1], c2 = co.c[s][2];
        double vq = 0.0, va = 0.0;
        if (on) l.U[ei][ej] = c2 * ns_dot<M>(l.A, l.A, ei, ej) + c1 * l.A[ei][ej] + (ei == ej ? c0 : 0.0);      // q
        __syncthreads();
        if (on) {
            vq = ns_dot<M>(l.U, l.Q, ei, ej);
            va = ns_dot<M>(l.U, l.A, ei, ej);
        }
        __syncthreads();
        if (on) {
            l.Q[ei][ej] = vq;
            l.V[ei][ej] = va;
        }
        __syncthreads();
        if (s + 1 < co.steps) {
            if (on) l.A[ei][ej] = ns_dot<M>(l.V, l.U, ei, ej);
            __syncthreads();
        }
    }
    fetch(0, false);
    for (int j0 = 0; j0 < n; j0 += JC) {
        __syncthreads();
        place();
        __syncthreads();
        if (j0 + JC < n) fetch(j0 + JC, false);
        float o[8];
#pragma unroll 2
        for (int q = 0; q < 8; ++q) {
            int i, j;
            place_of(tid + 256 * q, i, j);
            double s = 0.0;
#pragma unroll 8
            for (int k = 0; k < M; ++k) s = fma(l.Q[i][k], (double)l.x[k * LDX + j], s);
            o[q] = (float)s;
        }
        ns_store_n(a, d, b, o, [&](int q) { int i, j; place_of(tid + 256 * q, i, j); return i; }, [&](int q) { int i, j; place_of(tid + 256 * q, i, j); return j0 + j; });
    }
}

__global__ void __launch_bounds__(256) ns_norm_kernel(const NsTab a)
{
    __shared__ double red[4];
    ns_norm(a, blockIdx.x, red);
}

// ---- the first launch of a chunk: whole small matrices, and the sums of squares of the others
__global__ void __launch_bounds__(256) ns_first_kernel(const NsTab a, const NsCoef co, const int nsmall_wg)
{
    __shared__ NsSmallLds l;
    const int id = blockIdx.x;
    if (id < nsmall_wg) {
        const int k = ns_find(a.small, a.nsmall, id), mi = a.nbig + k, b = id - a.small[k], m = a.mat[mi].m;
        if (m <= 4) ns_small<4>(a, co, mi, b, l);
        else if (m <= 8) ns_small<8>(a, co, mi, b, l);
        else ns_small<16>(a, co, mi, b, l);
        return;
    }
    ns_norm(a, id - nsmall_wg, &l.A[0][0]);
}

inline int ns_pad(int v, int to) { return (v + to - 1) / to * to; }
inline int ns_short(const p2c_ns_matrix &m) { return m.rows < m.cols ? m.rows : m.cols; }
inline int ns_long(const p2c_ns_matrix &m) { return m.rows < m.cols ? m.cols : m.rows; }

// ns_small takes 9 us for small sides up to 8 and 64 columns, 12 for 5 x 500, 15 for 16 x 64, 31 for 16 x 512, 97 for 12 x 2000; the other forms take 27, 62, 27, 63
// and 82.
inline bool ns_is_small(const p2c_ns_matrix &m) { return ns_short(m) <= 8 || (ns_short(m) <= NS_SMALL && ns_long(m) <= 1024); }

// How a chunk is run.  Small matrices have a launch of their own - unless there are larger ones whose launches they can ride in: they lengthen none of their
// chains and leave the first launch to the norms (the 19 backbone matrices, three of them small: 158 -> 148 us; an optimizer step of theirs 161 -> 148).
// Batches stay: they would bring more tiles than the others have.
struct NsPlan { bool small[NS_MAX], mid; int tile; };           // mid: every one that is not small fits ns_mid_kernel

// Tile of a chunk's products: 128 keeps the matrix units busy (a wave reads 8 KB of operands for 12 instructions), 64 has four times the
// workgroups and a shorter chain per workgroup.  The choice is made for the widest product (all tiles); the padding of the sides follows it.  The symmetric
// products of a chunk on 128 take 128 x 64 (code 96), as they have half the tiles (8 x 1024 x 2048, 288 or 576 tiles: 81 and 48 us or 77 and 46; 2048 x 2048,
// 4000 x 1000, ...: 93 or 72).  256 x 128 with eight waves measured the same as 128 x 128 within 2 % both ways.
inline NsPlan ns_plan(const p2c_ns_matrix *mats, int n)
{
    NsPlan p;
    p.mid = true;
    auto fits = [](const p2c_ns_matrix &m) { return (long long)ns_pad(m.rows, 64) * ns_pad(m.cols, 64) <= NS_MID; };
    int longest = 0;
    for (int i = 0; i < n; ++i)
        if (!ns_is_small(mats[i]) && mats[i].batch) {
            longest = ns_long(mats[i]) > longest ? ns_long(mats[i]) : longest;
            p.mid = p.mid && fits(mats[i]);
        }
    long long t128 = 0;
    for (int i = 0; i < n; ++i) {
        p.small[i] = ns_is_small(mats[i]) && !(mats[i].batch == 1 && ns_long(mats[i]) <= longest && (!p.mid || fits(mats[i])));
        if (!p.small[i]) t128 += (long long)((mats[i].rows + 127) / 128) * ((mats[i].cols + 127) / 128) * mats[i].batch;
    }
    p.tile = !p.mid && t128 >= 256 ? 128 : 64;
    return p;
}

inline size_t ns_one_ws(const p2c_ns_matrix &m, int tile)
{
    const int mP = ns_pad(ns_short(m), tile), nP = ns_pad(ns_long(m), tile);
    return NS_PARTS * 8 + 3 * ns_xbytes(mP, nP) + 2 * ns_xbytes(mP, mP);
}

// sides up to 2^23 (the byte offset of a tile's rows in a block of 32 k has 32 bits), 65536 matrices per descriptor (a launch's workgroups)
int ns_check(const p2c_ns_matrix *mats, int n)
{
    if (!mats || n <= 0) return P2C_EINVAL;
    for (int i = 0; i < n; ++i)
        if (mats[i].rows < 0 || mats[i].cols < 0 || mats[i].batch < 0 || mats[i].rows > (1 << 23) || mats[i].cols > (1 << 23) ||
            (long long)mats[i].rows * mats[i].cols > (1ll << 31) || mats[i].batch > (1 << 16)) return P2C_EINVAL;
    return P2C_OK;
}

template <int TR, int TB, int KG, int NST, int PH>
int ns_product(const NsTab *tab, const NsRec *recs, int grid, float ca, float cb, int cur, hipStream_t st)
{
    constexpr int WG = ns_waves(TB), OUT = WG * 8192 + (KG == 1 ? 0 : KG * WG * 4 * 64 * 16), OPS = KG * (TR + TB) * 128 * NST,
                  LDS = OPS > OUT ? OPS : OUT;
    static_assert(LDS <= 160 * 1024, "");
    if (LDS > 65536) {
        const hipError_t rc = hipFuncSetAttribute((const void *)ns_product_kernel<TR, TB, KG, NST, PH>, hipFuncAttributeMaxDynamicSharedMemorySize, LDS);
        if (rc != hipSuccess) return (int)rc;
    }
    hipLaunchKernelGGL((ns_product_kernel<TR, TB, KG, NST, PH>), dim3(grid), dim3(64 * WG * KG), LDS, st, tab, recs, ca, cb, cur);
    P2C_LAUNCH_CHECK();
    return P2C_OK;
}

// The tile of one product of the chunk.  Few tiles: 32 with the k range shared by four waves - such a product is bound by the time its operands take
// to arrive, and this form has the most of them in flight over the most CUs (products of the 19 backbone matrices, 405 tiles of 32: 10.2 and 7.6 us
// against 14.0 and 9.0 with 64).  Many: it reads every operand twice as often (the decoder's seven 512 x 512, 988 tiles of 32: 20 us against 10).
inline int ns_pick(const NsTab &a, bool sym, int pad)
{
    long long t32 = 0;
    for (int i = 0; i < a.nbig; ++i) {
        const long long mt = a.mat[i].mP / 32, nt = a.mat[i].nP / 32;
        t32 += (sym ? mt * (mt + 1) / 2 : mt * nt) * a.mat[i].batch;
    }
    return pad == 128 ? (sym ? 96 : 128) : t32 <= 512 ? 32 : 64;
}

inline int ns_starts(NsTab &a, int phase, int tile)
{
    for (int i = 0; i < a.nbig; ++i) {
        const int tr = ns_tile_rows(tile), tb = ns_tile_cols(tile), m = a.mat[i].mP, n = a.mat[i].nP;
        a.start[phase][i + 1] = a.start[phase][i] + (phase == NS_SYM ? ns_sym_tiles(m, tr, tb) : (m / tb) * (n / tr)) * a.mat[i].batch;
    }
    return a.start[phase][a.nbig];
}

template <int PH>
int ns_product_any(const NsTab *tab, const NsRec *recs, int tile, int grid, float ca, float cb, int cur, hipStream_t st)
{
    if constexpr (PH <= 2) {
        if (tile == 96) return ns_product<128, 64, 1, 3, PH>(tab, recs, grid, ca, cb, cur, st);
    } else {
        if (tile == 128) return ns_product<128, 128, 1, 2, PH>(tab, recs, grid, ca, cb, cur, st);
    }
    if (tile == 64) return ns_product<64, 64, 1, 3, PH>(tab, recs, grid, ca, cb, cur, st);
    return ns_product<32, 32, 4, PH == 1 ? 3 : 2, PH>(tab, recs, grid, ca, cb, cur, st);
}

// the chunk's table (without ws); returns the bytes of workspace it needs
size_t ns_table(const p2c_ns_matrix *mats, int n, NsTab &a)
{
    const NsPlan plan = ns_plan(mats, n);
    const bool mid = plan.mid;
    const int tile = plan.tile;
    a.nbig = a.nsmall = 0;
    a.start[NS_NORM][0] = a.start[NS_TILES][0] = a.start[NS_SYM][0] = a.start[NS_ALL][0] = a.small[0] = 0;
    size_t off = 0;
    for (int small = 0; small < 2; ++small)
        for (int i = 0; i < n; ++i) {
            const p2c_ns_matrix &q = mats[i];
            if (!q.rows || !q.cols || !q.batch || (int)plan.small[i] != small) continue;
            NsMat &d = a.mat[a.nbig + a.nsmall];
            d.src = (const char *)q.src; d.mom = q.mom; d.dst = (char *)q.dst;
            d.src_rs = q.src_rs; d.src_cs = q.src_cs; d.src_bs = q.src_bs;
            d.dst_rs = q.dst_rs; d.dst_cs = q.dst_cs; d.dst_bs = q.dst_bs;
            d.tall = q.rows > q.cols;
            d.m = d.tall ? q.cols : q.rows; d.n = d.tall ? q.rows : q.cols;
            d.mP = ns_pad(d.m, tile); d.nP = ns_pad(d.n, tile);
            d.batch = q.batch; d.scale = q.scale; d.decay = q.decay;
            d.ws = off; d.ws_bs = small ? 0 : ns_one_ws(q, tile);
            off += d.ws_bs * q.batch;
            if (small) {
                a.small[a.nsmall + 1] = a.small[a.nsmall] + q.batch;
                ++a.nsmall;
            } else {
                const int j = a.nbig++;
                if (mid) a.start[NS_ALL][j + 1] = a.start[NS_ALL][j] + q.batch;
                a.start[NS_NORM][j + 1] = a.start[NS_NORM][j] + ns_parts(d.m, d.n) * q.batch;
                a.start[NS_TILES][j + 1] = a.start[NS_TILES][j] + (d.mP / 64) * (d.nP / 64) * q.batch;
            }
        }
    a.mid = mid;
    if (!a.nbig || mid) return 0;
    a.tsym = ns_pick(a, true, tile); a.tall = ns_pick(a, false, tile);
    a.nsym = ns_starts(a, NS_SYM, a.tsym); a.nall = ns_starts(a, NS_ALL, a.tall);
    const size_t head = ns_head(a.nsym, a.nall);
    for (int i = 0; i < a.nbig; ++i) a.mat[i].ws += head;
    return off + head;
}

int ns_chunk(const p2c_ns_matrix *mats, int n, int dtype, float mu, int muon, const NsCoef &co, double eps, char *ws, hipStream_t st)
{
    NsTab a;
    memset(&a, 0, sizeof a);
    a.ws = ws; a.dtype = dtype; a.mu = mu; a.muon = muon; a.eps = eps;
    ns_table(mats, n, a);
    if (!(a.nbig + a.nsmall)) return P2C_OK;
    // small matrices: in one launch with the sums of squares if those are few (the registers of ns_small leave two workgroups a CU)
    const int nsm = a.small[a.nsmall], nno = a.mid ? 0 : a.start[NS_NORM][a.nbig], apart = nno > 512 || !nsm;
    if (nsm) {
        hipLaunchKernelGGL(ns_first_kernel, dim3(nsm + (apart ? 0 : nno)), dim3(256), 0, st, a, co, nsm);
        P2C_LAUNCH_CHECK();
    }
    if (nno && apart) {
        hipLaunchKernelGGL(ns_norm_kernel, dim3(nno), dim3(256), 0, st, a);
        P2C_LAUNCH_CHECK();
    }
    if (!a.nbig) return P2C_OK;
    if (a.mid) {
        int most = 0;
        for (int i = 0; i < a.nbig; ++i) most = a.mat[i].mP * a.mat[i].nP > most ? a.mat[i].mP * a.mat[i].nP : most;
        const int lds = 2 * most * 4 + 64;
        const hipError_t rc = hipFuncSetAttribute((const void *)ns_mid_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 2 * NS_MID * 4 + 64);
        if (rc != hipSuccess) return (int)rc;
        hipLaunchKernelGGL(ns_mid_kernel, dim3(a.start[NS_ALL][a.nbig]), dim3(512), lds, st, a, co);
        P2C_LAUNCH_CHECK();
        return P2C_OK;
    }
    hipLaunchKernelGGL(ns_begin_kernel, dim3(a.start[NS_TILES][a.nbig]), dim3(256), 0, st, a);
    P2C_LAUNCH_CHECK();
    const NsTab *tab = (const NsTab *)ws;
    const NsRec *rsym = (const NsRec *)(ws + NS_TAB_BYTES), *rall = rsym + a.nsym;
    for (int s = 0; s < co.steps; ++s) {
        int rc = ns_product_any<1>(tab, rsym, a.tsym, a.nsym, 0.f, 1.f, s & 1, st);
        if (rc == P2C_OK) rc = ns_product_any<2>(tab, rsym, a.tsym, a.nsym, co.c[s][1], co.c[s][2], s & 1, st);
        if (rc == P2C_OK) rc = s + 1 < co.steps ? ns_product_any<3>(tab, rall, a.tall, a.nall, co.c[s][0], 1.f, s & 1, st)
                                                : ns_product_any<4>(tab, rall, a.tall, a.nall, co.c[s][0], 1.f, s & 1, st);
        if (rc != P2C_OK) return rc;
    }
    return P2C_OK;
}

int ns_run(const p2c_ns_matrix *mats, int n, int dtype, float mu, int muon, int steps, const float *coeffs, double eps, void *ws, size_t ws_bytes,
           void *stream)
{
    const int rc = ns_check(mats, n);
    if (rc != P2C_OK) return rc;
    if (steps < 1 || steps > 16 || !coeffs || !(eps > 0.0) || !isfinite(eps) || dtype < 0 || dtype > 2) return P2C_EINVAL;
    NsCoef co;
    co.steps = steps;
    // every matrix of the iteration has to stay inside the range of the scaled fp16 pairs: follow the bound of the spectrum
    double top = 1.0, gain[16];
    for (int s = 0; s < steps; ++s) {
        const double c0 = coeffs[3 * s], c1 = coeffs[3 * s + 1], c2 = coeffs[3 * s + 2];
        if (!isfinite(c0) || !isfinite(c1) || !isfinite(c2)) return P2C_EINVAL;
        double p = 0.0, q = 0.0;
        gain[s] = 0.0;
        for (int k = 0; k <= 64; ++k) {
            const double x = top * k / 64, t = x * x, bb = c1 * t + c2 * t * t, qq = c0 + bb;
            p = fmax(p, fabs(x * qq));
            q = fmax(q, fmax(fabs(bb), fabs(c0)));
            gain[s] = fmax(gain[s], fabs(qq));
        }
        if (!(p < 3.8) || !(q < 15.0)) return P2C_EINVAL;
        top = 1.01 * p;
        for (int k = 0; k < 3; ++k) co.c[s][k] = coeffs[3 * s + k];
    }
    double grown = 1.0;                                          // by the steps from s on: what the pairs drop at s
    for (int s = steps - 1; s >= 0; --s) {
        grown *= gain[s];
        if (!(grown <= 32768.0)) return P2C_EINVAL;
    }
    for (int s = steps; s < 16; ++s) co.c[s][0] = co.c[s][1] = co.c[s][2] = 0.f;
    for (int i = 0; i < n; ++i) {
        const p2c_ns_matrix &q = mats[i];
        if (q.rows && q.cols && q.batch && (!q.src || !q.dst || (muon && (!q.mom || q.batch != 1)))) return P2C_EINVAL;
    }
    size_t need = 0;
    NsTab tab;
    for (int i = 0; i < n; i += NS_MAX) {
        const size_t c = ns_table(mats + i, n - i < NS_MAX ? n - i : NS_MAX, tab);
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
    NsTab tab;
    for (int i = 0; i < n; i += NS_MAX) {
        const size_t c = ns_table(mats_host + i, n - i < NS_MAX ? n - i : NS_MAX, tab);
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
